"""Orders between the two CTAs of a pair, read from the kernels' sources: no
result shows on every run that one is missing.

A barrier operation that names no scope orders within its own CTA.  Arrivals at
the other CTA's barrier and the waits for them name the cluster; what shared
memory holds is released by the arrival and acquired by the wait."""
import glob
import os
import re

import pytest

from conftest import ROOT

CSRC = os.path.join(ROOT, "mlirpass_b200", "csrc")
SOURCES = {os.path.basename(p): open(p).read() for p in sorted(glob.glob(os.path.join(CSRC, "*.cu*")))}
SHARED = SOURCES["dcf_tensor.cuh"]
KERNELS = [name for name, text in SOURCES.items() if name != "dcf_tensor.cuh" and "arrive_first" in text]


def body(name: str) -> str:
    return re.search(r" %s\(uint64_t\* bar.*?\n}\n" % name, SHARED, re.S)[0]


def test_arrivals_at_the_other_ctas_barrier_name_the_cluster():
    arrivals = [a for text in SOURCES.values() for a in re.findall(r"mbarrier\.arrive\S*shared::cluster\S*", text)]
    assert arrivals
    for a in arrivals:
        assert ".release.cluster." in a or ".relaxed.cluster." in a, a


def test_what_is_published_is_released_and_acquired():
    publish, other = body("arrive_first").split("if constexpr (PUBLISH)")[1].split("else")
    assert ".release.cluster." in publish and ".relaxed.cluster." in other
    assert ".acquire.cluster." in body("pair_acquire")
    for name in ("pair_wait", "pair_wait_parked", "pair_test"):
        assert ".relaxed.cluster." in body(name)


@pytest.mark.parametrize("name", KERNELS)
def test_waits_are_their_arrivals_counterparts(name):
    text = SOURCES[name]
    arrivals = re.findall(r"arrive_first<(true|false)>\(&(\w+)\[", text)
    assert len(arrivals) == text.count("arrive_first")
    for publish, bar in arrivals:
        waits = set(re.findall(r"\b(\w+)\(&%s\[" % bar, text)) - {"mbar_init", "arrive_first"}
        allowed = {"pair_acquire"} if publish == "true" else {"pair_wait", "pair_wait_parked", "pair_test"}
        assert waits and waits <= allowed, (bar, waits)


@pytest.mark.parametrize("name", KERNELS)
def test_reads_of_tensor_memory_are_fenced_before_their_arrival(name):
    text = SOURCES[name]
    for at in re.finditer(r"arrive_first<false>", text):
        assert "tcgen05.fence::before_thread_sync" in text[at.start() - 200:at.start()]
