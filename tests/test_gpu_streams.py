"""Calls of the Python binding on a stream that is not the current one: what they
allocate is memory of that stream, whatever the current one still has queued."""
import pytest
import torch

pytestmark = pytest.mark.gpu
FP8, I8 = 3, 4


def cases(dev):
    """name -> call(stream) returning tensors that the call made."""
    from breeze_tts_cpp_amd import qlinear as q
    g = torch.Generator().manual_seed(12)
    bf = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(dev)
    M, N, K = 700, 1040, 1024
    x, big = bf(M, K), bf(8, 2 * K)
    wq, sw = q.row_quantize(bf(N, K), I8)
    xq, sx = q.row_quantize(x, I8)
    norm = bf(K)
    logits = torch.randn(4096, 64, generator=g).to(dev)
    ids = torch.randint(-1, 40, (9000,), generator=g, dtype=torch.int32).to(dev)
    few = torch.randint(0, 6, (M,), generator=g, dtype=torch.int32).to(dev)
    order, slots, offsets = q.group_rows(few, 6)
    W, SW = torch.stack([wq] * 6), torch.stack([sw] * 6)
    rows, rank = 4096, 64
    xa, a, b, base = bf(rows, 6144), bf(2, rank, 6144), bf(2, 256, rank), bf(rows, 256)
    a_order, _, a_offsets = q.group_rows((torch.arange(rows) % 2).int().to(dev), 2)
    assert q.adapter_workspace_bytes(rows, 2, 6144, rank) > 0
    split = q.Path(q.KIND_SKINNY, 16, 16, 4, 8)
    need = q.workspace_bytes(split, 8, N, 2 * K, I8)
    wq2, sw2 = q.row_quantize(bf(N, 2 * K), I8)
    xq2, sx2 = q.row_quantize(big, I8)
    assert need > 0
    xs, ws = x[:, :256].contiguous(), wq[:, :256].contiguous()
    # (What a caller hands over is made before, and ready on any stream.)
    own, own_r, y = torch.empty_like(ids), torch.empty(4096 * 8, dtype=torch.int32, device=dev), base.clone()
    return {
        "row_quantize": lambda s: q.row_quantize(x, I8, 128, 128, stream=s),
        "quantized_norm": lambda s: q.quantized_norm(x, norm, FP8, stream=s),
        "quantized_gated": lambda s: q.quantized_gated(x, I8, stream=s),
        "layer_norm_quantize": lambda s: q.layer_norm_quantize(x, I8, stream=s),
        "pointwise_quantize": lambda s: q.pointwise_quantize(x, I8, stream=s),
        "pointwise": lambda s: q.pointwise(x, stream=s),
        "norm_linear": lambda s: q.norm_linear(xs, ws, sw, I8, stream=s),
        "gemm": lambda s: q.gemm(xq, sx, wq, sw, I8, stream=s),
        "gemm_split": lambda s: q.gemm(xq2, sx2, wq2, sw2, I8, path=split, stream=s),
        "gemm_finish": lambda s: q.gemm_finish(xq2, sx2, wq2, sw2, I8, path=split, stream=s),
        "linear": lambda s: q.linear(x, wq, sw, I8, stream=s),
        "linear_noalloc": lambda s: q.linear_noalloc(x, wq, sw, I8, stream=s),
        "pack_weights": lambda s: q.pack_weights(wq, stream=s).data,
        "group_rows": lambda s: q.group_rows(ids, 40, stream=s),
        "group_rows_parts": lambda s: q.group_rows(ids, 40, order=own, stream=s)[1:],
        "route": lambda s: q.route(logits, 8, stream=s),
        "route_parts": lambda s: q.route(logits, 8, order=own_r, stream=s)[:2],
        "combine": lambda s: q.combine(x, slots.view(-1, 2), stream=s),
        "expert_gemm": lambda s: q.expert_gemm(xq, sx, W, SW, I8, offsets, order=order, scatter=True, stream=s),
        "adapter_add": lambda s: q.adapter_add(xa, a_order, a_offsets, a, b, y, base=base, stream=s),
    }


NAMES = ["row_quantize", "quantized_norm", "quantized_gated", "layer_norm_quantize", "pointwise_quantize",
         "pointwise", "norm_linear", "gemm", "gemm_split", "gemm_finish", "linear", "linear_noalloc", "pack_weights",
         "group_rows", "group_rows_parts", "route", "route_parts", "combine", "expert_gemm", "adapter_add"]


def tensors(result):
    return list(result) if isinstance(result, tuple) else [result]


def bits(t):
    return t.contiguous().view(torch.uint8).clone()


@pytest.fixture(scope="module")
def calls(dev):
    made = cases(dev)
    assert list(made) == NAMES
    return made


@pytest.mark.parametrize("name", [n for n in NAMES if n != "adapter_add"])  # (returns the caller's y)
@pytest.mark.parametrize("raw", [False, True])
def test_results_are_the_streams_memory(dev, calls, name, raw):
    """Blocks that the current stream has just freed are not what the call gets."""
    side = torch.cuda.Stream()
    torch.cuda.empty_cache()
    kept = tensors(calls[name](None))
    blocks = [(t.untyped_storage().data_ptr(), t.untyped_storage().nbytes()) for t in kept]
    torch.cuda.synchronize()
    del kept
    got = tensors(calls[name](side.cuda_stream if raw else side))
    torch.cuda.synchronize()
    for t in got:
        p = t.untyped_storage().data_ptr()
        assert not any(b <= p < b + n for b, n in blocks)


@pytest.mark.parametrize("name", NAMES)
def test_work_queued_on_the_current_stream(dev, calls, name):
    """The current stream is behind, its freed blocks still to be written; results
    that the caller drops at once are still being written on the other stream."""
    side = torch.cuda.Stream()
    want = [bits(t) for t in tensors(calls[name](None))]
    m = torch.randn(4096, 4096, device=dev)
    torch.cuda.synchronize()
    for _ in range(3):
        for _ in range(6):
            m = (m @ m).clamp_(-1, 1)  # the current stream is some ms behind
        # Every cached block of the usual sizes is freed with a write still to come.
        junk = [torch.full((1 << n,), 7, dtype=torch.int32, device=dev) for n in range(6, 23) for _ in range(2)]
        del junk
        result = tensors(calls[name](side))
        with torch.cuda.stream(side):
            got = [bits(t) for t in result]
            again = tensors(calls[name](None))
            later = [bits(t) for t in again]
        del result, again
        junk = [torch.full((1 << n,), 9, dtype=torch.int32, device=dev) for n in range(6, 23) for _ in range(2)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got)) and all(torch.equal(a, b) for a, b in zip(want, later))
        del junk, got, later


def test_the_current_stream_by_its_handle(dev, calls):
    """A stream argument that is the current one changes nothing."""
    from breeze_tts_cpp_amd import qlinear as q
    for name in ("gemm", "route", "expert_gemm"):
        want = [bits(t) for t in tensors(calls[name](None))]
        for s in (torch.cuda.current_stream(), torch.cuda.current_stream().cuda_stream):
            assert all(torch.equal(a, bits(t)) for a, t in zip(want, tensors(calls[name](s))))


def test_the_default_stream_from_another(dev, calls):
    """The default stream as the argument, by object and by its handle (0), while another is current."""
    here = torch.cuda.Stream()
    for name in ("linear", "route", "combine", "adapter_add"):
        want = [bits(t) for t in tensors(calls[name](None))]
        torch.cuda.synchronize()
        for s in (torch.cuda.default_stream(), 0):
            with torch.cuda.stream(here):
                got = tensors(calls[name](s))
            torch.cuda.synchronize()
            assert all(torch.equal(a, bits(t)) for a, t in zip(want, got)), name


@pytest.mark.parametrize("name", ["linear", "gemm_split", "route", "expert_gemm", "adapter_add"])
def test_forked_in_a_graph(dev, calls, name):
    """Captured on a stream that forks from the capturing one and joins it again; what the
    call makes lives in the graph's pool."""
    want = [bits(t) for t in tensors(calls[name](None))]
    main, fork = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        fork.wait_stream(main)
        first = tensors(calls[name](fork))
        second = tensors(calls[name](fork))
        main.wait_stream(fork)
    torch.cuda.synchronize()
    for _ in range(4):
        for t in first + second:
            t.zero_()
        junk = torch.full((1 << 20,), 5, dtype=torch.int32, device=dev)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for outs in (first, second):
            assert all(torch.equal(a, bits(t)) for a, t in zip(want, outs))
        del junk
