"""Quantized products of rows grouped by expert against plain 64-bit products:
INT8 per channel bit for bit, FP8 and K groups within a bound derived from the
sums (grouped_reference.expert_rows)."""
import numpy as np
import pytest
import torch

from tests import grouped_reference as ref

pytestmark = pytest.mark.gpu
FP8, I8 = 3, 4
MODES = {"int8": (I8, 0), "fp8": (FP8, 0), "group_int8": (I8, 128), "group_fp8": (FP8, 128)}
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def codes(g, rows, K, mode):
    fmt, group = MODES[mode]
    if fmt == I8:
        q = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8).view(torch.uint8)
    else:
        q = (100 * torch.randn(rows, K, generator=g)).clamp_(-448, 448).to(torch.float8_e4m3fn)
        q = q.view(torch.uint8)
    shape = (-(-K // group), rows) if group else (rows,)
    return q, (0.5 + torch.rand(*shape, generator=g)) * 0.01


def run_case(dev, mode, sizes, N, K, top_k=1, gather=True, scatter=False, dtype="bf16", path=None,
             absent=0, seed=0):
    """Experts with `sizes` rows each, `absent` ids without one; the whole output
    checked, rows without a group against their old contents."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(seed + N + K)
    fmt, group = MODES[mode]
    experts = len(sizes)
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(sizes)] + [torch.full((absent,), -1)])
    ids = ids[torch.randperm(ids.numel(), generator=g)].int()
    pad = -ids.numel() % top_k
    ids = torch.cat([ids, torch.full((pad,), -1, dtype=torch.int32)])
    count = ids.numel()
    order, _, offsets = ref.group(ids.numpy(), experts)
    rows = count // top_k if gather else count
    x, sx = codes(g, rows, K, mode)
    w, sw = zip(*[codes(g, N, K, mode) for _ in range(experts)])
    old = torch.randn(count, N, generator=g).to(DT[dtype])
    print(f"experts {mode} sizes={sizes} N={N} K={K} top_k={top_k} gather={gather} "
          f"scatter={scatter} {dtype} path={path}", flush=True)
    out = qlinear.expert_gemm(
        x.to(dev), sx.to(dev), torch.stack(w).to(dev), torch.stack(sw).to(dev), fmt,
        torch.from_numpy(offsets).to(dev), order=torch.from_numpy(order).to(dev) if gather else None,
        divisor=top_k, scatter=scatter, group=group, path=path, out=old.to(dev)).cpu()
    left = np.ones(count, bool)
    for e in range(experts):
        slots = np.arange(offsets[e], offsets[e + 1])
        if not slots.size:
            continue
        source = order[slots] // top_k if gather else slots
        to = order[slots] if scatter else slots
        left[to] = False
        sxe = sx[:, source] if group else sx[source]
        want = ref.expert_rows(x[source], sxe, w[e], sw[e], fmt, group, DT[dtype])
        if torch.is_tensor(want):
            assert torch.equal(out[to], want), f"expert {e}"
        else:
            assert torch.all((out[to].double() - want[0]).abs() <= want[1]), f"expert {e}"
    keep = torch.from_numpy(np.nonzero(left)[0])
    assert torch.equal(out[keep].view(torch.int16), old[keep].view(torch.int16))
    return out


def every_path():
    from breeze_tts_cpp_amd import qlinear
    seen = []
    for slots in (1, 64, 200, 2000, 6400, 12800, 20000, 40000, 100000):
        for K in (256, 2048, 4096):
            for mode, (fmt, group) in MODES.items():
                for N in (256, 1024, 2048, 4096):
                    for experts in (8, 64):
                        p = qlinear.expert_plan(slots, experts, N, K, fmt, group)
                        if (mode, p) not in seen:
                            seen.append((mode, p))
    assert len(seen) == 16  # five tiles per channel, three with K groups
    return seen


# Sizes around every tile height, odd K and N (past whole stages and tiles), empty
# experts first, last and between.
SIZES = [0, 1, 15, 0, 16, 17, 33, 64, 65, 0, 127, 130, 0]


@pytest.mark.parametrize("N,K", [(16, 16), (80, 144), (272, 656), (528, 1040)])
def test_every_tile(dev, N, K):
    for mode, path in every_path():
        run_case(dev, mode, SIZES, N, K, top_k=3, path=path, absent=9)


@pytest.mark.parametrize("K", [256, 384, 528])
def test_every_tile_whole(dev, K):
    """Whole and nearly whole tiles, few stages of K."""
    for mode, path in every_path():
        run_case(dev, mode, [256, 0, 257, 193], 272, K, top_k=2, path=path)


@pytest.mark.parametrize("mode", MODES)
def test_every_tile_repeats(dev, mode):
    """The same call gives the same bits, with every CU at work."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(17)
    fmt, group = MODES[mode]
    count, experts, N, K = 3000, 8, 1040, 1680
    ids = torch.randint(0, experts, (count,), generator=g, dtype=torch.int32).to(dev)
    x, sx = codes(g, count, K, mode)
    w, sw = codes(g, N, K, mode)
    x, sx, w = x.to(dev), sx.to(dev), torch.stack([w] * experts).to(dev)
    sw = torch.stack([sw] * experts).to(dev)
    order, _, offsets = qlinear.group_rows(ids, experts)
    for path in [p for m, p in every_path() if m == mode]:
        first = None
        for _ in range(6):
            out = qlinear.expert_gemm(x, sx, w, sw, fmt, offsets, order=order, scatter=True,
                                      group=group, path=path)
            first = out if first is None else first
            assert torch.equal(out, first), path


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gather,scatter", [(False, False), (True, False), (True, True)])
def test_planned(dev, mode, dtype, gather, scatter):
    run_case(dev, mode, [3, 0, 40, 1, 7, 0], 272, 2048, 2 if gather and not scatter else 1, gather,
             scatter, dtype, absent=5)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("sizes,N,K", [([1], 16, 32), ([0, 0, 1, 0], 2064, 2048), ([300], 256, 512),
                                       ([600, 0, 5], 512, 384), ([2] * 100, 48, 128),
                                       ([1, 0] * 300, 32, 64), ([520, 530], 768, 6144)])
def test_planned_shapes(dev, mode, sizes, N, K):
    run_case(dev, mode, sizes, N, K, top_k=1, absent=2)


@pytest.mark.parametrize("mode", MODES)
def test_nothing_chosen(dev, mode):
    """No id names an expert: no row is written."""
    run_case(dev, mode, [0, 0, 0], 64, 128, absent=40)


def test_row_does_not_depend_on_its_place(dev):
    """The same rows and experts in another order of rows give the same bits."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(5)
    for mode, (fmt, group) in MODES.items():
        count, experts, N, K = 500, 6, 320, 1040
        ids = torch.randint(0, experts, (count,), generator=g, dtype=torch.int32)
        x, sx = codes(g, count, K, mode)
        w, sw = zip(*[codes(g, N, K, mode) for _ in range(experts)])
        w, sw = torch.stack(w).to(dev), torch.stack(sw).to(dev)
        perm = torch.randperm(count, generator=g)
        outs = []
        for p in (torch.arange(count), perm):
            order, _, offsets = qlinear.group_rows(ids[p].to(dev), experts)
            sxp = sx[:, p].contiguous() if group else sx[p]
            outs.append(qlinear.expert_gemm(x[p].to(dev), sxp.to(dev), w, sw, fmt, offsets,
                                            order=order, scatter=True, group=group).cpu())
        assert torch.equal(outs[0][perm], outs[1]), mode


def test_far_expert(dev):
    """An expert whose weights start past 4 GiB."""
    from breeze_tts_cpp_amd import qlinear
    experts, N, K = 520, 4096, 2064  # 4.4 GB of codes
    g = torch.Generator().manual_seed(1)
    w = torch.zeros(experts, N, K, dtype=torch.uint8, device=dev)
    sw = torch.zeros(experts, N, device=dev)
    wl, swl = codes(g, N, K, "int8")
    w[-1], sw[-1] = wl.to(dev), swl.to(dev)
    x, sx = codes(g, 3, K, "int8")
    ids = torch.tensor([experts - 1, 0, experts - 1], dtype=torch.int32, device=dev)
    order, _, offsets = qlinear.group_rows(ids, experts)
    y = qlinear.expert_gemm(x.to(dev), sx.to(dev), w, sw, I8, offsets, order=order, scatter=True).cpu()
    want = ref.expert_rows(x[[0, 2]], sx[[0, 2]], wl, swl, I8, 0, torch.bfloat16)
    assert torch.equal(y[[0, 2]], want) and torch.all(y[1] == 0)


def test_bad_indices_stay_in_bounds(dev):
    """Offsets past the slots or descending, and order entries outside the rows:
    such rows count as zeros or are dropped, the others keep their values."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(9)
    x, sx = codes(g, 8, 128, "int8")
    w, sw = codes(g, 32, 128, "int8")
    W, SW = torch.stack([w, w, w]).to(dev), torch.stack([sw, sw, sw]).to(dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    full = ref.expert_rows(x, sx, w, sw, I8, 0, torch.bfloat16)
    out = torch.zeros(8, 32, dtype=torch.bfloat16, device=dev)
    qlinear.expert_gemm(x.to(dev), sx.to(dev), W, SW, I8, i32([-5, 4, 2, 1000]), out=out)
    assert torch.equal(out.cpu(), full)
    out = torch.zeros(8, 32, dtype=torch.bfloat16, device=dev)
    order = i32([3, -1, 8, 2**31 - 1, -2**31, 0, 7, 1])
    qlinear.expert_gemm(x.to(dev), sx.to(dev), W, SW, I8, i32([0, 8, 8, 8]), order=order,
                        scatter=True, out=out)
    want = torch.zeros_like(full)
    for r in (3, 0, 7, 1):
        want[r] = full[r]
    assert torch.equal(out.cpu(), want)


# (offsets, slots): each held to [0, slots] and to the largest before it, as numpy does it below.
@pytest.mark.parametrize("offsets,slots", [([-5, 4, 2, 1000], 8), ([0, 6, 1, 8, 3, 8], 8),
                                           ([40, 3, 20, 70, 60, 75], 70), ([0] * 30 + [9, 2] * 20 + [33], 33),
                                           ([64, 0] * 70 + [90], 90)])
def test_a_slot_has_one_expert(dev, offsets, slots):
    """Offsets out of order or out of range: a slot that several experts claim is the
    first one's, one that none claims keeps what it held, on every tile."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(len(offsets))
    experts, N, K = len(offsets) - 1, 80, 144
    held = np.maximum.accumulate(np.clip(offsets, 0, slots))
    for mode, path in every_path():
        fmt, group = MODES[mode]
        x, sx = codes(g, slots, K, mode)
        w, sw = zip(*[codes(g, N, K, mode) for _ in range(experts)])
        old = torch.randn(slots, N, generator=g).to(torch.bfloat16)
        print(f"experts {mode} offsets={offsets} slots={slots} path={path}", flush=True)
        out = qlinear.expert_gemm(x.to(dev), sx.to(dev), torch.stack(w).to(dev), torch.stack(sw).to(dev), fmt,
                                  torch.tensor(offsets, dtype=torch.int32, device=dev), group=group, path=path,
                                  out=old.to(dev)).cpu()
        left = np.ones(slots, bool)
        for e in range(experts):
            at = np.arange(held[e], held[e + 1])
            if not at.size:
                continue
            left[at] = False
            want = ref.expert_rows(x[at], sx[:, at] if group else sx[at], w[e], sw[e], fmt, group, torch.bfloat16)
            if torch.is_tensor(want):
                assert torch.equal(out[at], want), (mode, path, e)
            else:
                assert torch.all((out[at].double() - want[0]).abs() <= want[1]), (mode, path, e)
        assert torch.equal(out[left].view(torch.int16), old[left].view(torch.int16))
