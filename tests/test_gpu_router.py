"""Router, grouping and return of rows against plain 64-bit forms."""
import numpy as np
import pytest
import torch

from tests import grouped_reference as ref

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def check_grouping(ids, groups, order, slots, offsets):
    want = ref.group(ids.cpu().numpy(), groups)
    for name, got, exp in zip(("order", "slots", "offsets"), (order, slots, offsets), want):
        assert np.array_equal(got.cpu().numpy().reshape(-1), exp), name


# (count, groups): one id, around a wave, one workgroup's most and one more,
# several runs, a last run of one id.
@pytest.mark.parametrize("count,groups", [(1, 1), (1, 1024), (63, 5), (64, 64), (65, 65), (1000, 3),
                                          (1025, 1024), (4096, 31), (4097, 128), (6145, 1000),
                                          (40000, 7), (140000, 513)])
def test_group_rows(dev, count, groups):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(count)
    ids = torch.randint(-2, groups + 2, (count,), generator=g, dtype=torch.int32)
    print(f"group_rows count={count} groups={groups}", flush=True)
    check_grouping(ids, groups, *qlinear.group_rows(ids.to(dev), groups))


@pytest.mark.parametrize("ids", [[-1] * 70, [2] * 70, [0, 2, 0, 2] * 20, [2, 1, 0], [2**31 - 1, -2**31, 1]])
def test_group_rows_one_sided(dev, ids):
    from breeze_tts_cpp_amd import qlinear
    t = torch.tensor(ids, dtype=torch.int32)
    check_grouping(t, 3, *qlinear.group_rows(t.to(dev), 3))
    t = t.repeat(400)  # the form for many ids
    check_grouping(t, 3, *qlinear.group_rows(t.to(dev), 3))


def check_route(qlinear, logits, top_k, normalize, **kw):
    ids, weights, order, slots, offsets = qlinear.route(logits, top_k, normalize, **kw)
    experts = logits.shape[1]
    v = logits.double().cpu().numpy()
    want_ids, want = ref.route(v, top_k, normalize)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    # Relative: the difference to the maximum is rounded (|d| half steps of 2^-23 at
    # most 104 before the exponential is 0), the exponential is off by a unit, a sum
    # of `experts` terms by one unit each, the division by half a one.
    rel = (104 + experts + 4) * 2.0 ** -23
    got = weights.double().cpu().numpy()
    assert np.all(np.abs(got - want) <= rel * want + 2.0 ** -126)
    check_grouping(ids, experts, order, slots, offsets)
    return ids, weights, order, slots, offsets


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("tokens,experts,top_k,normalize",
                         [(1, 1, 1, True), (1, 8, 2, False), (5, 16, 16, True), (16, 17, 4, False),
                          (64, 64, 6, True), (33, 65, 8, False), (40, 128, 8, True),
                          (16, 129, 16, False), (9, 256, 3, True), (7, 1000, 16, False),
                          (70, 60, 2, True), (1100, 32, 4, False)])
def test_route(dev, dtype, tokens, experts, top_k, normalize):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(tokens * 1000 + experts)
    v = 3 * torch.randn(tokens, experts + 3, generator=g)
    v[torch.rand(v.shape, generator=g) < 0.05] = float("-inf")
    v = v.to(DT[dtype]).to(dev)
    print(f"route {dtype} tokens={tokens} experts={experts} top_k={top_k}", flush=True)
    check_route(qlinear, v[:, :experts], top_k, normalize)  # a row stride past the experts


@pytest.mark.parametrize("experts", [4, 100, 300])
def test_route_values(dev, experts):
    """Ties, signed zeros, rows with nothing left, infinities, NaN, the lowest and
    largest values: the first index wins, NaN and -inf are never chosen."""
    from breeze_tts_cpp_amd import qlinear
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    rows = torch.zeros(12, experts)
    rows[1, :] = -inf
    rows[2, :] = nan
    rows[3, :] = -inf
    rows[3, 2] = low
    rows[4, 1:4] = inf
    rows[5, 0], rows[5, 3] = -0.0, 0.0
    rows[6, :] = nan
    rows[6, 1], rows[6, 3] = -7.0, -7.0
    rows[7, :] = low
    rows[8, 3] = -low
    rows[9, 0] = 1e-45
    rows[10, :] = torch.arange(experts) % 2
    rows[11, 1] = -1e-45
    for top_k in (1, 3, 4):
        for normalize in (False, True):
            check_route(qlinear, rows.to(dev), top_k, normalize)
            check_route(qlinear, rows.repeat(120, 1).to(dev), top_k, normalize)


def test_route_many_tokens(dev):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(3)
    v = torch.randn(2051, 48, generator=g).to(torch.bfloat16).to(dev)
    first = check_route(qlinear, v, 8, True)
    again = qlinear.route(v, 8, True)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


# N: whole rows, odd sizes, more than one 2048-column tile.
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,top_k,N,base", [(1, 1, 8, False), (3, 2, 1, True), (16, 6, 2048, False),
                                                 (5, 16, 2056, True), (37, 3, 777, True),
                                                 (2, 4, 4099, False), (130, 8, 256, True)])
def test_combine(dev, dtype, tokens, top_k, N, base):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(tokens + N)
    rows = tokens * top_k + 2
    h = torch.randn(rows, N, generator=g).to(DT[dtype])
    slots = torch.randint(-1, rows, (tokens, top_k), generator=g, dtype=torch.int32)
    slots[0, 0] = rows  # past the rows: left out
    w = torch.randn(tokens, top_k, generator=g)
    unread = sorted(set(range(rows)) - set(slots.flatten().tolist()))
    h[unread] = float("nan")  # rows that no slot names are not read
    b = torch.randn(tokens, N, generator=g).to(DT[dtype]) if base else None
    print(f"combine {dtype} tokens={tokens} top_k={top_k} N={N}", flush=True)
    for weights in (w, None):
        want = torch.zeros(tokens, N, dtype=torch.float64) if b is None else b.double()
        size = want.abs()
        for t in range(tokens):
            for j in range(top_k):
                if 0 <= slots[t, j] < rows:
                    term = h[slots[t, j]].double() * (1.0 if weights is None else float(weights[t, j]))
                    want[t] += term
                    size[t] += term.abs()
        got = qlinear.combine(h.to(dev), slots.to(dev), None if weights is None else weights.to(dev),
                              base=None if b is None else b.to(dev)).double().cpu()
        # top_k fma and one addition, each half a step of a partial sum; the result's rounding.
        bound = (top_k + 1) * 2.0 ** -24 * size + ref.HALF_STEP[DT[dtype]] * (want.abs() + 2.0 ** -20 * size)
        assert torch.all((got - want).abs() <= bound + torch.finfo(DT[dtype]).tiny)


def test_combine_in_place_and_empty(dev):
    """out may be base; a token whose slots are all absent keeps its base (0 without one)."""
    from breeze_tts_cpp_amd import qlinear
    h = torch.full((4, 64), float("nan"), dtype=torch.bfloat16, device=dev)
    slots = torch.full((3, 2), -1, dtype=torch.int32, device=dev)
    base = torch.randn(3, 64, device=dev).to(torch.bfloat16)
    keep = base.clone()
    out = qlinear.combine(h, slots, torch.ones(3, 2, device=dev), base=base, out=base)
    assert out.data_ptr() == base.data_ptr() and torch.equal(out, keep)
    assert torch.equal(qlinear.combine(h, slots), torch.zeros_like(keep))
