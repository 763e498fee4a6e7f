"""Forms of the operators on grouped rows that sizes, types and alignments select
beside the usual ones: 16-bit types and stores of every tile, the router past what
one table of counts holds, 16-bit logits of special values, special codes and scales,
and calls with workspaces captured and at the same time."""
import numpy as np
import pytest
import torch

from tests import grouped_reference as ref
from tests.test_gpu_experts import MODES, SIZES, codes, every_path
from tests.test_gpu_grouped_layer import Layer, inputs, same
from tests.test_gpu_router import check_route

pytestmark = pytest.mark.gpu
FP8, I8 = 3, 4
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------- expert products
# (top_k 1: scatter to the rows; shift: the output's first element, 8-byte steps.)
@pytest.mark.parametrize("dtype,scatter,shift", [("f16", True, 0), ("f16", False, 4), ("bf16", True, 4),
                                                 ("f16", True, 12)])
@pytest.mark.parametrize("N,K", [(80, 144), (272, 656)])
def test_every_tile_stores(dev, dtype, scatter, shift, N, K):
    """Every tile's results in both types, in slot order and scattered, on and off 16 bytes."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(N + shift)
    experts, dt = len(SIZES), DT[dtype]
    ids = torch.cat([torch.full((n,), e) for e, n in enumerate(SIZES)] + [torch.full((9,), -1)])
    ids = ids[torch.randperm(ids.numel(), generator=g)].int()
    count = ids.numel()
    order, _, offsets = ref.group(ids.numpy(), experts)
    for mode, path in every_path():
        fmt, group = MODES[mode]
        x, sx = codes(g, count, K, mode)
        w, sw = zip(*[codes(g, N, K, mode) for _ in range(experts)])
        old = torch.randn(count * N + shift + 8, generator=g).to(dt)
        held = old.to(dev)
        out = held[shift:shift + count * N].view(count, N)
        assert out.data_ptr() % 16 == shift * 2 % 16
        print(f"experts {mode} {dtype} scatter={scatter} shift={shift} N={N} K={K} path={path}", flush=True)
        qlinear.expert_gemm(x.to(dev), sx.to(dev), torch.stack(w).to(dev), torch.stack(sw).to(dev), fmt,
                            torch.from_numpy(offsets).to(dev), order=torch.from_numpy(order).to(dev),
                            scatter=scatter, group=group, path=path, out=out)
        got = held.cpu()
        want = old.clone()
        rows, wrows = got[shift:shift + count * N].view(count, N), want[shift:shift + count * N].view(count, N)
        for e in range(experts):
            slots = np.arange(offsets[e], offsets[e + 1])
            if not slots.size:
                continue
            src = order[slots]
            to = src if scatter else slots
            y = ref.expert_rows(x[src], sx[:, src] if group else sx[src], w[e], sw[e], fmt, group, dt)
            if torch.is_tensor(y):
                assert torch.equal(rows[to], y), (mode, path, e)
            else:
                assert torch.all((rows[to].double() - y[0]).abs() <= y[1]), (mode, path, e)
            wrows[to] = rows[to]
        assert torch.equal(got.view(torch.int16), want.view(torch.int16))  # nothing else written


@pytest.mark.parametrize("mode", MODES)
def test_special_codes_and_scales(dev, mode):
    """A NaN code, a zero, infinite or NaN scale of a row, a channel or a K group reaches
    its own row or channel alone; INT8 -128 is a value like others. On every tile."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(31)
    fmt, group = MODES[mode]
    sizes, N, K = [40, 0, 70, 130], 144, 400
    experts, count = len(sizes), sum(sizes)
    offsets = torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32).to(dev)
    of = torch.repeat_interleave(torch.arange(experts), torch.tensor(sizes))
    x, sx = codes(g, count, K, mode)
    w, sw = zip(*[codes(g, N, K, mode) for _ in range(experts)])
    w, sw = torch.stack(w), torch.stack(sw)
    if fmt == I8:
        x[5], w[2, 7] = 0x80, 0x80  # -128 throughout
    call = lambda path, *t: qlinear.expert_gemm(*(v.to(dev) for v in t), fmt, offsets, group=group, path=path).cpu()
    # Rows 3 (inf), 44 (NaN), 111 (0) by their scale, row 60 by a code; channels 9 of
    # expert 0 (NaN), 20 of 2 (0), 143 of 3 (inf) by their scale, 77 of 3 by a code.
    x2, sx2, w2, sw2 = x.clone(), sx.clone(), w.clone(), sw.clone()
    at = (lambda r: (0, r)) if group else (lambda r: (r,))       # K group 0 alone
    last = (lambda r: (-1, r)) if group else (lambda r: (r,))    # the last, short one
    sx2[at(3)], sx2[last(44)] = float("inf"), float("nan")
    sx2[..., 111] = 0.0
    sw2[(0, *at(9))], sw2[(3, *last(143))] = float("nan"), float("inf")
    sw2[2, ..., 20] = 0.0
    if fmt == FP8:
        x2[60, 399], w2[3, 77, 130] = 0x7f, 0xff
    for path in [p for m, p in every_path() if m == mode]:
        print(f"special {mode} path={path}", flush=True)
        clean, got = call(path, x, sx, w, sw), call(path, x2, sx2, w2, sw2)
        if fmt == I8 and not group:
            for e in range(experts):
                mine = of == e
                if mine.any():
                    assert torch.equal(clean[mine], ref.expert_rows(x[mine], sx[mine], w[e], sw[e], I8, 0,
                                                                    torch.bfloat16))
                    want = ref.expert_rows(x2[mine], sx2[mine], w2[e], sw2[e], I8, 0, torch.bfloat16)
                    assert torch.equal(got[mine].isnan(), want.isnan())
                    assert torch.equal(got[mine].nan_to_num(), want.nan_to_num())
        odd = torch.zeros(count, N, dtype=torch.bool)
        odd[3], odd[44], odd[111] = True, True, True
        odd[of == 0, 9], odd[of == 2, 20], odd[of == 3, 143] = True, True, True
        if fmt == FP8:
            odd[60], odd[of == 3, 77] = True, True
            assert got[60].isnan().all() and got[of == 3, 77].isnan().all()
        assert torch.equal(got[~odd], clean[~odd])
        assert got[44].isnan().all() and got[of == 0, 9].isnan().all()
        assert not got[3].isfinite().any() and not got[of == 3, 143].isfinite().any()  # (0 * inf is NaN)
        zero = torch.ones(N, dtype=torch.bool)
        zero[[77, 143] if fmt == FP8 else [143]] = False
        assert torch.all(got[111, zero] == 0)
        rest = of == 2
        rest[[44, 60] if fmt == FP8 else [44]] = False
        assert torch.all(got[rest, 20] == 0)


# ---------------------------------------------------------------- router
@pytest.mark.parametrize("dtype,tokens,experts,top_k", [("bf16", 16385, 64, 2), ("f32", 4097, 256, 3),
                                                        ("f16", 4097, 200, 2), ("f32", 16390, 16, 1)])
def test_route_past_the_table(dev, dtype, tokens, experts, top_k):
    """More workgroups than the table of counts has rows."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(tokens)
    v = torch.randn(tokens, experts, generator=g).to({"f32": torch.float32, **DT}[dtype])
    v[torch.rand(v.shape, generator=g) < 0.02] = float("-inf")
    print(f"route {dtype} tokens={tokens} experts={experts}", flush=True)
    check_route(qlinear, v.to(dev), top_k, True)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("experts", [4, 100, 300])
def test_route_values_16_bit(dev, dtype, experts):
    """Ties, signed zeros, infinities, NaN, the lowest, largest and smallest values of the type."""
    from breeze_tts_cpp_amd import qlinear
    dt = DT[dtype]
    inf, nan, info = float("inf"), float("nan"), torch.finfo(dt)
    rows = torch.zeros(14, experts, dtype=dt)
    rows[1, :] = -inf
    rows[2, :] = nan
    rows[3, :] = -inf
    rows[3, 2] = info.min
    rows[4, 1:4] = inf
    rows[5, 0], rows[5, 3] = -0.0, 0.0
    rows[6, :] = nan
    rows[6, 1], rows[6, 3] = -7.0, -7.0
    rows[7, :] = info.min
    rows[8, 3] = info.max
    rows[9, 0] = info.smallest_normal * info.eps  # the least subnormal
    rows[10, :] = torch.arange(experts) % 2
    rows[11, 1] = -info.smallest_normal * info.eps
    rows[12, :] = torch.tensor(1.0) + info.eps * (torch.arange(experts) % 3)  # neighbours
    rows[13, :] = -(torch.tensor(1.0) + info.eps * (torch.arange(experts) % 3))
    assert rows[9, 0] > 0 and rows[11, 1] < 0
    for top_k in (1, 3, 4):
        for normalize in (False, True):
            check_route(qlinear, rows.to(dev), top_k, normalize)
            check_route(qlinear, rows.repeat(120, 1).to(dev), top_k, normalize)


# ---------------------------------------------------------------- workspaces
def large_layer(dev, mode):
    """More than 4096 choices, and adapters in their two launches."""
    from breeze_tts_cpp_amd import qlinear
    layer = Layer(dev, mode, 2304, hidden=1024, adapters=3, rank=128)
    assert qlinear.adapter_workspace_bytes(2304, 3, 1024, 128) > 0
    return layer


@pytest.mark.parametrize("mode", ["int8", "group_fp8"])
def test_workspaces_in_graphs(dev, mode):
    """Two captured steps, each with workspaces of its own, replayed at once."""
    layer = large_layer(dev, mode)
    steps = []
    for i in range(2):
        held, o, stream = inputs(dev, layer, i), layer.buffers(dev), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            layer.run(*held, o, stream=stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run(*held, o, stream=stream)
        steps.append((held, o, stream, graph))
    for replay in range(3):
        print(f"workspaces graph {mode} replay {replay}", flush=True)
        for i, (held, o, _, _) in enumerate(steps):
            for t, new in zip(held, inputs(dev, layer, 50 + 10 * replay + i, padded=replay * 100)):
                t.copy_(new)
            for name in ("gu", "down"):
                o[name].zero_()
        torch.cuda.synchronize()
        for _, _, stream, graph in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for held, o, _, _ in steps:
            eager = layer.run(*held, layer.buffers(dev))
            torch.cuda.synchronize()
            wrong = [k for k, v in same(o, eager).items() if not v]
            assert not wrong, (replay, wrong)


def test_workspaces_on_two_streams(dev):
    """Eager steps on two streams at once, their workspaces made by the calls."""
    layer = large_layer(dev, "int8")
    held = [inputs(dev, layer, i) for i in range(2)]
    want = [layer.run(*h, layer.buffers(dev)) for h in held]
    got, streams = [layer.buffers(dev) for _ in held], [torch.cuda.Stream() for _ in held]
    torch.cuda.synchronize()
    for _ in range(6):
        for h, o, s in zip(held, got, streams):
            with torch.cuda.stream(s):
                layer.run(*h, o)
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(same(w, o).values())


def test_given_workspaces(dev):
    """Workspaces of the caller, of exactly the size needed and with whatever they held."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(3000, 48, generator=g).to(dev)
    ids = torch.randint(-1, 200, (70001,), generator=g, dtype=torch.int32).to(dev)
    rows, K, rank, N = 2304, 1024, 128, 144
    x, y0 = torch.randn(rows, K, generator=g).half().to(dev), torch.randn(rows, N, generator=g).half().to(dev)
    a, b = (torch.randn(2, rank, K, generator=g) / 32).half().to(dev), torch.randn(2, N, rank, generator=g).half().to(dev)
    order, _, offsets = qlinear.group_rows((torch.arange(rows) % 2).int().to(dev), 2)
    need = [qlinear.load().qlin_group_rows_workspace_bytes(6000, 48),
            qlinear.load().qlin_group_rows_workspace_bytes(70001, 200),
            qlinear.adapter_workspace_bytes(rows, 2, K, rank)]
    assert min(need) > 0
    run = lambda ws: (*qlinear.route(logits, 2, workspace=ws[0]), *qlinear.group_rows(ids, 200, workspace=ws[1]),
                      qlinear.adapter_add(x, order, offsets, a, b, torch.empty_like(y0), base=y0, workspace=ws[2]))
    want = run([None] * 3)
    # 64 bytes past each that must stay as they are.
    whole = [torch.full((n + 64,), 0xff, dtype=torch.uint8, device=dev) for n in need]
    for fill in (0xff, 0x7f, 0):
        for t in whole:
            t.fill_(fill)
        got = run([t[:n] for t, n in zip(whole, need)])
        assert all(torch.equal(p, q) for p, q in zip(want, got))
        assert all(torch.all(t[n:] == fill) for t, n in zip(whole, need))
    for i in range(3):
        short = [t[:n - 1] if i == j else t[:n] for j, (t, n) in enumerate(zip(whole, need))]
        with pytest.raises(qlinear.QLinearError):
            run(short)
