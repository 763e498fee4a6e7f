"""The operators on grouped rows together, as a serving step runs them: a
mixture layer (router, codes, gathered products, gate, products, return onto a
shared projection with its requests' adapters) and codebook heads. Every stage
is checked against its 64-bit form on the inputs that it had, and captured steps
against eager ones bit for bit, with other requests in every replay."""
import numpy as np
import pytest
import torch

from tests import grouped_reference as ref

pytestmark = pytest.mark.gpu
FP8, I8 = 3, 4
MODES = {"int8": (I8, 0, 0), "fp8": (FP8, 0, 0), "group_int8": (I8, 128, 128), "group_fp8": (FP8, 128, 128)}


class Layer:
    """hidden -> top_k of `experts` (gate | up, SiLU, down), a shared projection and
    adapters of `rank` per request; buffers for up to `tokens` rows."""

    def __init__(self, dev, mode, tokens, seed=0, hidden=256, inter=384, experts=6, top_k=2, adapters=3,
                 rank=16):
        from breeze_tts_cpp_amd import qlinear as q
        g = torch.Generator().manual_seed(seed)
        bf = lambda *s, sc=1.0: (sc * torch.randn(*s, generator=g)).to(torch.bfloat16).to(dev)
        self.q, self.mode, self.tokens, self.top_k, self.experts = q, mode, tokens, top_k, experts
        self.fmt, self.group, self.rot = MODES[mode]
        self.hidden, self.inter, self.adapters = hidden, inter, adapters

        def quantized(n, k):
            parts = [q.row_quantize(bf(n, k, sc=k ** -0.5), self.fmt, self.group, self.rot)
                     for _ in range(experts)]
            return torch.stack([c for c, _ in parts]), torch.stack([s for _, s in parts])

        self.w1, self.s1 = quantized(2 * inter, hidden)
        self.w2, self.s2 = quantized(hidden, inter)
        self.shared_w, self.shared_s = q.row_quantize(bf(hidden, hidden, sc=hidden ** -0.5), I8)
        self.a, self.b = bf(adapters, rank, hidden, sc=hidden ** -0.5), bf(adapters, hidden, rank, sc=0.2)
        self.scales = torch.rand(adapters, generator=g).to(dev)
        self.router = (torch.randn(hidden, experts, generator=g) * hidden ** -0.5).to(dev)

    def buffers(self, dev):
        t, k, h, n = self.tokens, self.top_k, self.hidden, self.tokens * self.top_k
        blocks = lambda c: (-(-c // self.group), n) if self.group else (n,)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)
        bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=dev)
        u8 = lambda *s: torch.zeros(*s, dtype=torch.uint8, device=dev)
        f32 = lambda *s: torch.zeros(*s, device=dev)
        tb = (-(-h // self.group), t) if self.group else (t,)
        return dict(ids=i32(t, k), weights=f32(t, k), order=i32(n), slots=i32(t, k), offsets=i32(self.experts + 1),
                    xq=u8(t, h), sx=f32(*tb), gu=bf(n, 2 * self.inter), aq=u8(n, self.inter),
                    sa=f32(*blocks(self.inter)), down=bf(n, h), shared=bf(t, h), out=bf(t, h),
                    sq=u8(t, h), ss=f32(t), a_order=i32(t), a_slots=i32(t), a_offsets=i32(self.adapters + 1))

    def run(self, x, logits, voices, o, stream=None):
        q, fmt, group, rot = self.q, self.fmt, self.group, self.rot
        q.route(logits, self.top_k, True, ids=o["ids"], weights=o["weights"], order=o["order"],
                slots=o["slots"], offsets=o["offsets"], stream=stream)
        q.row_quantize(x, fmt, group, rot, values=o["xq"], scales=o["sx"], stream=stream)
        q.expert_gemm(o["xq"], o["sx"], self.w1, self.s1, fmt, o["offsets"], order=o["order"],
                      divisor=self.top_k, group=group, out=o["gu"], stream=stream)
        q.quantized_gated(o["gu"], fmt, 0, group, rot, values=o["aq"], scales=o["sa"], stream=stream)
        q.expert_gemm(o["aq"], o["sa"], self.w2, self.s2, fmt, o["offsets"], group=group, out=o["down"],
                      stream=stream)
        q.linear(x, self.shared_w, self.shared_s, I8, scratch=(o["sq"], o["ss"]), out=o["shared"],
                 stream=stream)
        q.group_rows(voices, self.adapters, order=o["a_order"], slots=o["a_slots"],
                     offsets=o["a_offsets"], stream=stream)
        q.adapter_add(x, o["a_order"], o["a_offsets"], self.a, self.b, o["shared"], scales=self.scales,
                      stream=stream)
        q.combine(o["down"], o["slots"], o["weights"], base=o["shared"], out=o["out"], stream=stream)
        return o


def inputs(dev, layer, seed, padded=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(layer.tokens, layer.hidden, generator=g).to(torch.bfloat16)
    logits = x.float() @ layer.router.cpu() + 0.1 * torch.randn(layer.tokens, layer.experts, generator=g)
    voices = torch.randint(-1, layer.adapters, (layer.tokens,), generator=g, dtype=torch.int32)
    if padded:  # rows behind the last request: no expert, no voice
        logits[-padded:] = float("-inf")
        voices[-padded:] = -1
    return x.to(dev), logits.to(dev), voices.to(dev)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("tokens,padded", [(1, 0), (19, 3), (300, 44)])
def test_layer(dev, mode, tokens, padded):
    layer = Layer(dev, mode, tokens)
    x, logits, voices = inputs(dev, layer, 11, padded)
    print(f"layer {mode} tokens={tokens}", flush=True)
    o = {k: v.cpu() for k, v in layer.run(x, logits, voices, layer.buffers(dev)).items()}
    x, logits, voices = x.cpu(), logits.cpu(), voices.cpu()
    k, fmt, group = layer.top_k, layer.fmt, layer.group
    ids, weights = ref.route(logits.double().numpy(), k, True)
    assert np.array_equal(o["ids"].numpy(), ids)
    rel = (104 + layer.experts + 4) * 2.0 ** -23
    assert np.all(np.abs(o["weights"].double().numpy() - weights) <= rel * weights)
    order, slots, offsets = ref.group(ids, layer.experts)
    for name, want in (("order", order), ("slots", slots), ("offsets", offsets)):
        assert np.array_equal(o[name].numpy().reshape(-1), want), name
    w = [t.cpu() for t in (layer.w1, layer.s1, layer.w2, layer.s2)]
    for e in range(layer.experts):
        at = np.arange(offsets[e], offsets[e + 1])
        if not at.size:
            continue
        src = order[at] // k
        for got, xq, sx, rows, wq, sw in ((o["gu"], o["xq"], o["sx"], src, w[0][e], w[1][e]),
                                          (o["down"], o["aq"], o["sa"], at, w[2][e], w[3][e])):
            want = ref.expert_rows(xq[rows], sx[:, rows] if group else sx[rows], wq, sw, fmt, group,
                                   torch.bfloat16)
            if torch.is_tensor(want):
                assert torch.equal(got[at], want)
            else:
                assert torch.all((got[at].double() - want[0]).abs() <= want[1])
    assert torch.all(o["gu"][offsets[-1]:] == 0) and torch.all(o["down"][offsets[-1]:] == 0)
    shared = layer.q.linear(x.to(dev), layer.shared_w, layer.shared_s, I8).cpu()
    for v in range(layer.adapters):
        at = torch.nonzero(voices == v).flatten()
        want, bound = ref.adapter_rows(x[at], layer.a[v].cpu(), layer.b[v].cpu(), shared[at],
                                       float(layer.scales[v]))
        assert torch.all((o["shared"][at].double() - want).abs() <= bound)
    none = torch.nonzero(voices < 0).flatten()
    assert torch.equal(o["shared"][none], shared[none])
    want, size = o["shared"].double(), o["shared"].double().abs()
    for t in range(tokens):
        for j in range(k):
            if o["slots"][t, j] >= 0:
                term = float(o["weights"][t, j]) * o["down"][o["slots"][t, j]].double()
                want[t] += term
                size[t] += term.abs()
    bound = (k + 1) * 2.0 ** -24 * size + 2.0 ** -8 * (want.abs() + 2.0 ** -20 * size)
    assert torch.all((o["out"].double() - want).abs() <= bound)


def same(a, b):
    return {k: torch.equal(a[k].view(torch.uint8) if a[k].dtype != torch.uint8 else a[k],
                           b[k].view(torch.uint8) if b[k].dtype != torch.uint8 else b[k]) for k in a}


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("tokens", [24, 300])
def test_layer_in_graphs(dev, mode, tokens):
    """Two steps captured with their own buffers, replayed on two streams at once
    with other requests each time; eager work between."""
    layer = Layer(dev, mode, tokens)
    steps = []
    for i in range(2):
        held, o = inputs(dev, layer, i), layer.buffers(dev)
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            layer.run(*held, o, stream=stream)  # eager first call
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            layer.run(*held, o, stream=stream)
        steps.append((held, o, stream, graph))
    for replay in range(4):
        print(f"layer graph {mode} tokens={tokens} replay {replay}", flush=True)
        for i, (held, o, stream, graph) in enumerate(steps):
            for t, new in zip(held, inputs(dev, layer, 100 + 10 * replay + i, padded=replay * tokens // 8)):
                t.copy_(new)
            for name in ("gu", "down"):
                o[name].zero_()  # rows of no expert keep what was there
        torch.cuda.synchronize()
        for held, o, stream, graph in steps:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for held, o, _, _ in steps:
            eager = layer.run(*held, layer.buffers(dev))
            torch.cuda.synchronize()
            wrong = [k for k, v in same(o, eager).items() if not v]
            assert not wrong, (replay, wrong)


def test_two_streams_at_once(dev):
    """Eager steps on two streams, nothing shared but the weights."""
    layer = Layer(dev, "int8", 200)
    held = [inputs(dev, layer, i) for i in range(2)]
    want = [layer.run(*h, layer.buffers(dev)) for h in held]
    got = [layer.buffers(dev) for _ in held]
    streams = [torch.cuda.Stream() for _ in held]
    torch.cuda.synchronize()
    for _ in range(8):
        for h, o, s in zip(held, got, streams):
            with torch.cuda.stream(s):
                layer.run(*h, o)  # the current stream
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(same(w, o).values())


def test_workspace_on_another_stream(dev):
    """Calls that make their workspace, on a stream that is not the current one."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(4)
    logits = torch.randn(4096, 64, generator=g).to(dev)
    rows, K, rank, N = 4096, 6144, 64, 256
    x = torch.randn(rows, K, generator=g).to(torch.bfloat16).to(dev)
    a, b = (torch.randn(2, rank, K, generator=g) / 80).to(torch.bfloat16).to(dev), \
        torch.randn(2, N, rank, generator=g).to(torch.bfloat16).to(dev)
    order, _, offsets = qlinear.group_rows((torch.arange(rows) % 2).int().to(dev), 2)
    base = torch.zeros(rows, N, dtype=torch.bfloat16, device=dev)
    want = [t.clone() for t in qlinear.route(logits, 8)]
    want_y = qlinear.adapter_add(x, order, offsets, a, b, torch.empty_like(base), base=base)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        got = qlinear.route(logits, 8, stream=side)
        y = qlinear.adapter_add(x, order, offsets, a, b, torch.empty_like(base), base=base, stream=side)
        junk = [torch.full((1 << 18,), 7, dtype=torch.int32, device=dev) for _ in range(4)]  # current stream
        torch.cuda.synchronize()
        assert all(torch.equal(p, r) for p, r in zip(want, got)) and torch.equal(y, want_y)
        del junk


@pytest.mark.parametrize("mode", ["int8", "group_fp8"])
def test_heads(dev, mode):
    """Rows at different codebooks through their own heads, back in request order."""
    from breeze_tts_cpp_amd import qlinear
    fmt, group, rot = MODES[mode]
    g = torch.Generator().manual_seed(7)
    rows, heads, N, K = 77, 31, 208, 256
    x = torch.randn(rows, K, generator=g).to(torch.bfloat16).to(dev)
    at = torch.randint(0, heads, (rows,), generator=g, dtype=torch.int32).to(dev)
    parts = [qlinear.row_quantize((torch.randn(N, K, generator=g) / 16).to(torch.bfloat16).to(dev), fmt, group, rot)
             for _ in range(heads)]
    w, sw = torch.stack([c for c, _ in parts]), torch.stack([s for _, s in parts])
    xq, sx = qlinear.row_quantize(x, fmt, group, rot)
    order, _, offsets = qlinear.group_rows(at, heads)
    y = qlinear.expert_gemm(xq, sx, w, sw, fmt, offsets, order=order, scatter=True, group=group).cpu()
    for r in range(rows):
        want = ref.expert_rows(xq[r:r + 1].cpu(), (sx[:, r:r + 1] if group else sx[r:r + 1]).cpu(),
                               w[at[r]].cpu(), sw[at[r]].cpu(), fmt, group, torch.bfloat16)
        if torch.is_tensor(want):
            assert torch.equal(y[r:r + 1], want)
        else:
            assert torch.all((y[r:r + 1].double() - want[0]).abs() <= want[1])


def test_rows_past_4_gib(dev):
    """Results and returned rows whose offsets pass 32 bits."""
    from breeze_tts_cpp_amd import qlinear
    g = torch.Generator().manual_seed(3)
    rows, N, K = (1 << 20) + 40, 2064, 16  # 4.3 GB of results
    ids = torch.full((rows,), -1, dtype=torch.int32)
    live = torch.tensor([0, 5, rows - 2, rows - 1])
    ids[live] = 0
    order, slots, offsets = qlinear.group_rows(ids.to(dev), 1)
    x = torch.randint(-127, 128, (rows, K), generator=g, dtype=torch.int8).view(torch.uint8)
    sx = torch.rand(rows, generator=g)
    w = torch.randint(-127, 128, (1, N, K), generator=g, dtype=torch.int8).view(torch.uint8)
    sw = torch.rand(1, N, generator=g)
    y = torch.zeros(rows, N, dtype=torch.bfloat16, device=dev)
    qlinear.expert_gemm(x.to(dev), sx.to(dev), w.to(dev), sw.to(dev), I8, offsets, order=order,
                        scatter=True, out=y)
    want = ref.expert_rows(x[live], sx[live], w[0], sw[0], I8, 0, torch.bfloat16)
    assert torch.equal(y[live.to(dev)].cpu(), want)
    back = qlinear.combine(y, torch.tensor([[rows - 1, 5], [-1, rows - 2]], dtype=torch.int32, device=dev))
    bound = 2.0 ** -8
    assert torch.allclose(back[1].float().cpu(), want[2].float(), rtol=0, atol=0)
    both = want[3].double() + want[1].double()
    assert torch.all((back[0].double().cpu() - both).abs() <= bound * both.abs() + 1e-30)


def test_operands_off_the_gpu(dev):
    from breeze_tts_cpp_amd import qlinear
    ids = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError):
        qlinear.group_rows(ids, 2)
    with pytest.raises(ValueError):
        qlinear.group_rows(ids.to(dev), 2, order=torch.zeros(8, dtype=torch.int32))
    with pytest.raises(ValueError):
        qlinear.route(torch.zeros(4, 8), 2)
    h = torch.zeros(8, 16, dtype=torch.bfloat16, device=dev)
    with pytest.raises(ValueError):
        qlinear.combine(h, torch.zeros(2, 2, dtype=torch.int32))
