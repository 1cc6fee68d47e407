"""The restated cuts against the workspaces that the library asks for, and what the sizes of the GPU tests reach."""
import random

import int8_cuts as cuts
import mlirpass_b200 as m


def sizes(seed: int, count: int):
    rng = random.Random(seed)
    for _ in range(count):
        yield tuple(int(2 ** rng.uniform(0, top)) for top in (13, 13, 13))


def test_products_ask_for_the_workspaces_of_their_cuts():
    parts = set()
    for tokens, channels, depth in sizes(1, 1500):
        for a_dtype, pad in (("i8", 0), ("bf16", 0), ("i8", 3), ("f32", 16)):
            plan = m.int8_matmul_plan(tokens, channels, depth, a_dtype=a_dtype, b_row_stride=depth + pad)
            assert plan.workspace == cuts.matmul_workspace(tokens, channels, depth, a_dtype == "i8", depth + pad), (tokens, channels, depth)
        if not cuts.few_tokens(tokens, depth):
            tn, _, n = cuts.matmul_cut(tokens, channels, depth)
            parts.add((tn, n > 1))
    assert len(parts) == 6, parts


def test_gradients_ask_for_the_workspaces_of_their_cuts():
    parts = set()
    for tokens, channels, depth in sizes(2, 1500):
        for pad in (0, 8, 3):
            plan = m.checkpoint_grad_plan("bf16", tokens, channels, depth, grad_row_stride=channels + pad)
            assert plan.workspace == cuts.grad_workspace(tokens, channels, depth, channels + pad), (tokens, channels, depth)
        tn, _, n = cuts.grad_cut(tokens, channels, depth)
        parts.add((tn, n > 1))
    assert len(parts) == 4, parts


def test_columns_before_a_gradient_take_no_more_than_is_asked_for():
    """Its cut with any number of them is the one with none or the one with seven."""
    for tokens, channels, depth in [*sizes(3, 500), *((t, c, d) for t in (100, 1000, 6000) for c in range(120, 137) for d in (40, 300, 1000))]:
        room = cuts.grad_workspace(tokens, channels, depth, -(-channels // 8) * 8 + 8)
        for skip in range(8):
            tn, tiles, parts = cuts.grad_cut(tokens, channels, depth, skip)
            assert cuts._room(tokens * -(-depth // 16) * 32, tiles * parts * 256 * tn * 4 if parts > 1 else 0) <= room
