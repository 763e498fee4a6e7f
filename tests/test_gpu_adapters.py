"""Low-rank adapters of many requests against plain 64-bit products, within a
bound derived from the sums (grouped_reference.adapter_rows)."""
import numpy as np
import pytest
import torch

from tests import grouped_reference as ref

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def run_case(dev, rows, adapters, rank, N, K, dtype, ranks=None, scales=True, base="y", xpad=0, ypad=0,
             absent=0.2, runs=1, spread=1.0, seed=0):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(seed + rows + N)
    dt = DT[dtype]
    rand = lambda *s: torch.randn(*s, generator=g)
    ids = torch.randint(0, adapters, (-(-rows // runs),), generator=g).repeat_interleave(runs)[:rows]
    ids[torch.rand(rows, generator=g) < absent] = -1
    order, _, offsets = ref.group(ids.numpy(), adapters)
    wide = (spread * rand(rows, K + xpad)).to(dt)
    a, b = (rand(adapters, rank, K) / K ** 0.5).to(dt), (rand(adapters, N, rank) / rank ** 0.5).to(dt)
    sc = 0.5 + torch.rand(adapters, generator=g) if scales else None
    used = [rank] * adapters
    if ranks is not None:
        used = [min(max(r, 0), rank) for r in ranks]
        for i, r in enumerate(used):  # what lies past a rank is not used
            a[i, r:], b[i, :, r:] = float("nan"), float("inf")
    y = rand(rows, N + ypad).to(dt)
    separate = rand(rows, N + ypad).to(dt)
    print(f"adapters rows={rows} adapters={adapters} rank={rank} N={N} K={K} {dtype} ranks={ranks} "
          f"xpad={xpad} ypad={ypad} base={base}", flush=True)
    yd, sd = y.to(dev), separate.to(dev)
    out = qlinear.adapter_add(
        wide.to(dev)[:, xpad:], torch.from_numpy(order).to(dev), torch.from_numpy(offsets).to(dev),
        a.to(dev), b.to(dev), yd[:, ypad:], base=None if base == "y" else sd[:, ypad:],
        ranks=None if ranks is None else torch.tensor(ranks, dtype=torch.int32, device=dev),
        scales=None if sc is None else sc.to(dev))
    assert out.data_ptr() == yd[:, ypad:].data_ptr()
    got, want = yd.cpu(), y.clone()
    start = y if base == "y" else separate
    for i in range(adapters):
        at = torch.from_numpy(np.nonzero(ids.numpy() == i)[0])
        if not at.numel():
            continue
        r = used[i]
        ref_y, bound = ref.adapter_rows(wide[at, xpad:], a[i, :r], b[i, :, :r], start[at, ypad:],
                                        1.0 if sc is None else float(sc[i]))
        far = (got[at, ypad:].double() - ref_y).abs()
        assert torch.all(far <= bound), (i, r, float((far / bound).max()))
        want[at, ypad:] = got[at, ypad:]
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))  # nothing else written


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rank", [1, 4, 8, 12, 16, 24, 32, 40, 64, 96, 100, 128])
def test_ranks(dev, dtype, rank):
    run_case(dev, 37, 5, rank, 144, 272, dtype)
    run_case(dev, 200, 3, rank, 144, 272, dtype, runs=20)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,adapters,N,K", [(1, 1, 16, 16), (1, 8, 4096, 2048), (2, 1, 32, 48),
                                               (16, 16, 2048, 2048), (17, 1, 272, 6144),
                                               (57, 70, 528, 1040), (64, 3, 4096, 160),
                                               (65, 2, 528, 1040), (129, 200, 144, 2048),
                                               (431, 6, 2064, 1024), (1000, 1, 256, 512)])
def test_shapes(dev, dtype, rows, adapters, N, K):
    run_case(dev, rows, adapters, 16, N, K, dtype)
    run_case(dev, rows, adapters, 16, N, K, dtype, absent=0.0, runs=7)


@pytest.mark.parametrize("rows", [40, 150])
@pytest.mark.parametrize("rank", [16, 12])
@pytest.mark.parametrize("xpad,ypad", [(8, 0), (0, 16), (3, 1), (16, 7), (1, 0)])
def test_strides(dev, rows, rank, xpad, ypad):
    run_case(dev, rows, 4, rank, 112, 208, "bf16", xpad=xpad, ypad=ypad)
    run_case(dev, rows, 4, rank, 112, 208, "f16", xpad=xpad, ypad=ypad, base="separate")


@pytest.mark.parametrize("rows", [30, 300])
def test_ragged_ranks(dev, rows):
    """Ranks of 0 (base alone), in between, and outside [0, rank] (held to it);
    what lies past a rank holds NaN and infinities."""
    run_case(dev, rows, 8, 64, 160, 320, "bf16", ranks=[0, 1, 7, 8, 33, 64, 99, -3])
    run_case(dev, rows, 8, 64, 160, 320, "f16", ranks=[64, 63, 31, 32, 0, 5, 16, 17], scales=False,
             base="separate")


@pytest.mark.parametrize("rows", [20, 100])
@pytest.mark.parametrize("spread", [1e-6, 3e4])
def test_inner_product_range(dev, rows, spread):
    """f16: the inner product far outside f16's range, large and small."""
    g = torch.Generator().manual_seed(2)
    from breeze_tts_cpp_amd import qlinear
    K, N, rank = 512, 64, 16
    x = (spread * (0.5 + torch.rand(rows, K, generator=g))).to(torch.float16)
    a = torch.rand(1, rank, K, generator=g).to(torch.float16)  # sums of K positive terms
    b = (torch.randn(1, N, rank, generator=g)).to(torch.float16)
    scale = 1.0 / (spread * K)
    y = torch.zeros(rows, N, dtype=torch.float16)
    order, offsets = torch.arange(rows, dtype=torch.int32), torch.tensor([0, rows], dtype=torch.int32)
    got = qlinear.adapter_add(x.to(dev), order.to(dev), offsets.to(dev), a.to(dev), b.to(dev), y.to(dev),
                              scales=torch.tensor([scale], device=dev)).cpu()
    want, bound = ref.adapter_rows(x, a[0], b[0], y, float(torch.tensor(scale)))
    assert torch.all((got.double() - want).abs() <= bound)


@pytest.mark.parametrize("rows", [20, 100])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_infinite_and_nan_rows(dev, rows, dtype):
    """An infinity or NaN in one row's x reaches that row alone."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(4)
    K, N, rank, dt = 96, 48, 8, DT[dtype]
    x = torch.randn(rows, K, generator=g).to(dt)
    a, b = torch.rand(1, rank, K, generator=g).to(dt), torch.rand(1, N, rank, generator=g).to(dt)
    y = torch.randn(rows, N, generator=g).to(dt)
    order = torch.arange(rows, dtype=torch.int32).to(dev)
    offsets = torch.tensor([0, rows], dtype=torch.int32, device=dev)
    call = lambda xx: qlinear.adapter_add(xx.to(dev), order, offsets, a.to(dev), b.to(dev), y.to(dev)).cpu()
    clean = call(x)
    x2 = x.clone()
    x2[3, 5], x2[11, 0] = float("inf"), float("nan")
    got = call(x2)
    keep = [r for r in range(rows) if r not in (3, 11)]
    assert torch.equal(got[keep], clean[keep])
    assert torch.all(got[3] == float("inf")) and torch.all(got[11].isnan())


def test_bad_indices_stay_in_bounds(dev):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(6)
    for rows in (8, 80):
        x, y = (torch.randn(rows, 64, generator=g).to(torch.bfloat16) for _ in range(2))
        a, b = (torch.randn(2, 8, 64, generator=g).to(torch.bfloat16),
                torch.randn(2, 64, 8, generator=g).to(torch.bfloat16))
        order = torch.arange(rows, dtype=torch.int32)
        offsets = torch.tensor([0, rows, rows], dtype=torch.int32)
        call = lambda o, f: qlinear.adapter_add(x.to(dev), o.to(dev), f.to(dev), a.to(dev), b.to(dev),
                                                y.to(dev)).cpu()
        full = call(order, offsets)
        assert torch.equal(call(order, torch.tensor([-9, 1 << 30, 5], dtype=torch.int32)), full)
        bad = order.clone()
        bad[0], bad[1], bad[2] = -1, rows, 2**31 - 1
        got = call(bad, offsets)
        assert torch.equal(got[3:], full[3:]) and torch.equal(got[:3], y[:3])


def test_row_does_not_depend_on_its_place(dev):
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(8)
    for rows in (50, 400):
        x, y = (torch.randn(rows, 256, generator=g).to(torch.bfloat16) for _ in range(2))
        a, b = (torch.randn(4, 16, 256, generator=g).to(torch.bfloat16).to(dev),
                torch.randn(4, 256, 16, generator=g).to(torch.bfloat16).to(dev))
        ids = torch.randint(0, 4, (rows,), generator=g, dtype=torch.int32)
        perm = torch.randperm(rows, generator=g)
        outs = []
        for p in (torch.arange(rows), perm):
            order, _, offsets = qlinear.group_rows(ids[p].to(dev), 4)
            outs.append(qlinear.adapter_add(x[p].to(dev), order, offsets, a, b, y[p].to(dev)).cpu())
        assert torch.equal(outs[0][perm], outs[1])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("rows,adapters,rank,N,K", [(2300, 3, 40, 272, 6160), (4096, 6, 64, 528, 4096),
                                                    (1500, 40, 128, 144, 4112), (6000, 2, 16, 96, 6144)])
def test_two_launches(dev, dtype, rows, adapters, rank, N, K):
    """Sizes of the form with a workspace, ranks off the 8, one adapter short of rows."""
    from breeze_tts_cpp_amd import qlinear
    assert qlinear.adapter_workspace_bytes(rows, adapters, K, rank) > 0
    run_case(dev, rows, adapters, rank, N, K, dtype, runs=rows // (adapters * 2) + 1)
    run_case(dev, rows, adapters, rank, N, K, dtype, runs=7, xpad=3, ypad=1, base="separate",
             ranks=[rank, 0, rank // 2 + 1] + [3] * (adapters - 3) if adapters > 2 else [rank, 5])


@pytest.mark.parametrize("offsets,rows,rank,N,K", [([-5, 4, 2, 1000], 8, 8, 64, 64),
                                                   ([40, 3, 20, 70, 60, 75], 70, 24, 80, 144),
                                                   ([0] * 30 + [9, 2] * 20 + [33], 33, 16, 48, 48),
                                                   ([100, 2000, 700, 3000, 5000], 2300, 40, 48, 6160)])
def test_a_row_has_one_adapter(dev, offsets, rows, rank, N, K):
    """Offsets out of order or out of range: a row that several adapters claim is the
    first one's, one that none claims keeps what it held (the last case: two launches)."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(rows)
    n = len(offsets) - 1
    held = np.maximum.accumulate(np.clip(offsets, 0, rows))
    x, y = torch.randn(rows, K, generator=g).to(torch.bfloat16), torch.randn(rows, N, generator=g).to(torch.bfloat16)
    a = (torch.randn(n, rank, K, generator=g) / K ** 0.5).to(torch.bfloat16)
    b = (torch.randn(n, N, rank, generator=g) / rank ** 0.5).to(torch.bfloat16)
    print(f"adapters offsets={offsets} rows={rows}", flush=True)
    got = qlinear.adapter_add(x.to(dev), torch.arange(rows, dtype=torch.int32, device=dev),
                              torch.tensor(offsets, dtype=torch.int32, device=dev), a.to(dev), b.to(dev),
                              y.to(dev)).cpu()
    left = np.ones(rows, bool)
    for i in range(n):
        at = np.arange(held[i], held[i + 1])
        if at.size:
            left[at] = False
            want, bound = ref.adapter_rows(x[at], a[i], b[i], y[at], 1.0)
            assert torch.all((got[at].double() - want).abs() <= bound), i
    assert torch.equal(got[left].view(torch.int16), y[left].view(torch.int16))
