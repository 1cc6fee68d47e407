"""How the 8-bit product and the gradient from a checkpoint cut their work, restated from the kernels' cost rules, so
that a test can say which of them it reaches.  The workspace sizes that the library reports depend on the cut."""
from math import ceil

PAIRS, SIDE, RUN = 74, 256, 128


def _least(costs):
    best = None
    for cost, cut in costs:
        if best is None or cost < best[0]:
            best = cost, cut
    return best[1]


def matmul_cut(tokens: int, channels: int, depth: int):
    """(tokens of a tile, tiles, parts of the depth) of a product of more than few tokens."""
    blocks = ceil(depth / 256)

    def costs():
        for tn, stage in ((64, 0.5), (128, 0.65), (256, 1)):
            tiles = ceil(channels / SIDE) * ceil(tokens / tn)
            s = 1
            while s == 1 or (s <= blocks and tiles * s <= PAIRS):
                each = ceil(blocks / s)
                parts = ceil(blocks / each) if each else 1
                yield ceil(tiles * parts / PAIRS) * each * stage + (5 if parts > 1 else 0) + 4 * stage, (tn, tiles, parts)
                s += 1
    return _least(costs())


def few_tokens(tokens: int, depth: int) -> bool:
    bucket = 1 if tokens <= 1 else 2 if tokens <= 2 else 4
    return tokens <= 4 and depth > 0 and bucket * (ceil(depth / 512) * 512 + 512) <= 64 << 10


def _room(*parts: int) -> int:
    return sum(ceil(p / 256) * 256 for p in parts)


def matmul_workspace(tokens: int, channels: int, depth: int, ints: bool, b_stride: int = 0) -> int:
    stride = ceil(depth / 16) * 16
    if few_tokens(tokens, depth):
        own = ints or tokens * depth <= 8192
        return 0 if own else _room(tokens * stride, tokens * 4)
    tn, tiles, parts = matmul_cut(tokens, channels, depth)
    copied = tn > 64 and channels > 1 and (b_stride or depth) % 16
    return _room(tokens * stride, 0 if ints else tokens * 4, channels * stride if copied else 0,
                 tiles * parts * SIDE * tn * 4 if parts > 1 else 0)


def grad_cut(tokens: int, channels: int, depth: int, skip: int = 0):
    """(channels of a tile, tiles, parts of the runs) of a gradient that starts `skip` elements into a vector."""
    runs = ceil(tokens / RUN)

    def costs():
        for tn, run in ((128, 0.65), (256, 1)):
            tiles = ceil(depth / SIDE) * ceil((channels + skip) / tn)
            s = 1
            while s == 1 or (s <= runs and tiles * s <= PAIRS):
                each = ceil(runs / s)
                parts = ceil(runs / each)
                yield ceil(tiles * parts / PAIRS) * (each + 5) * run + (6 if parts > 1 else 0), (tn, tiles, parts)
                s += 1
    return _least(costs())


def grad_workspace(tokens: int, channels: int, depth: int, grad_stride: int = 0) -> int:
    if not tokens or not channels or not depth:
        return 0
    stride = grad_stride or channels
    copied = tokens > 1 and (stride % 8 or stride < channels)

    def one(skip):
        tn, tiles, parts = grad_cut(tokens, channels, depth, skip)
        return _room(tokens * ceil(depth / 16) * 32, tokens * ceil(channels / 8) * 16 if copied else 0,
                     tiles * parts * SIDE * tn * 4 if parts > 1 else 0)
    return one(0) if copied else max(one(0), one(7))
