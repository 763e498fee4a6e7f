"""Refusals of the operators on grouped rows, without a GPU: every call below
fails its checks before anything reaches the device."""
import ctypes

import pytest
import torch

from breeze_tts_cpp_amd import qlinear

BF16, F32, I32, FP8, I8, F16 = 0, 1, 2, 3, 4, 5
FAKE = 0x10000  # never dereferenced
FAR = 0x40000000000
# Addresses far apart, for arrays that must not overlap.
IDS, ORDER, SLOTS, OFFSETS, WEIGHTS = (FAR * k for k in range(2, 7))


def test_group_rows_refusals():
    L = qlinear.load()

    def call(ids=IDS, count=100, groups=8, order=ORDER, slots=SLOTS, offsets=OFFSETS, ws=None, wsb=0):
        return L.qlin_group_rows(ids, count, groups, order, slots, offsets, ws, wsb, None)

    assert call(count=0) == -1 and call(count=(1 << 30) + 1) == -1
    assert call(groups=0) == -1 and call(groups=1025) == -1
    for name in ("ids", "order", "slots", "offsets"):
        assert call(**{name: None}) == -1
        assert call(**{name: FAKE + 2}) == -2
    assert call(slots=IDS) == -1 and b"overlap" in L.qlin_last_error()
    assert call(order=IDS + 396) == -1 and call(offsets=SLOTS - 32) == -1
    need = L.qlin_group_rows_workspace_bytes(100000, 8)
    assert need > 0 and L.qlin_group_rows_workspace_bytes(4096, 1024) == 0
    assert call(count=100000) == -3 and b"workspace" in L.qlin_last_error()
    assert call(count=100000, ws=FAKE, wsb=need - 1) == -3
    assert call(count=100000, ws=FAKE + 2, wsb=need) == -2
    assert L.qlin_group_rows_workspace_bytes(0, 8) == 0
    assert L.qlin_group_rows_workspace_bytes(10, 2000) == 0


def test_route_refusals():
    L = qlinear.load()

    def call(logits=FAKE, ld=64, t=F32, tokens=4, experts=64, k=2, ids=IDS, w=WEIGHTS, order=ORDER,
             slots=SLOTS, off=OFFSETS, ws=None, wsb=0):
        return L.qlin_route(logits, ld, t, tokens, experts, k, 0, ids, w, order, slots, off, ws, wsb,
                            None)

    assert call(t=I8) == -1 and call(tokens=0) == -1 and call(experts=0) == -1
    assert call(experts=1025, ld=1025) == -1 and call(ld=63) == -1
    assert call(k=0) == -1 and call(k=17) == -1 and call(experts=3, k=4) == -1
    for name in ("logits", "ids", "w", "order", "slots", "off"):
        assert call(**{name: None}) == -1
    assert call(logits=FAKE + 2) == -2 and call(w=WEIGHTS + 2) == -2
    assert call(w=FAKE + 4) == -1 and call(ids=FAKE + 1020) == -1 and call(w=SLOTS) == -1
    assert call(t=BF16, logits=FAKE + 1) == -2
    assert call(tokens=4096, k=2) == -3
    assert call(tokens=1 << 29, k=8) == -1  # more choices than an index holds


def test_combine_refusals():
    L = qlinear.load()

    def call(h=FAKE, rows=8, slots=FAKE, w=FAKE, base=None, out=FAR, tokens=4, k=2, N=64, t=BF16):
        return L.qlin_combine(h, rows, slots, w, base, out, tokens, k, N, t, None)

    assert call(t=F32) == -1 and call(rows=0) == -1 and call(tokens=0) == -1
    assert call(k=0) == -1 and call(k=17) == -1 and call(N=0) == -1
    for name in ("h", "slots", "out"):
        assert call(**{name: None}) == -1
    assert call(h=FAKE + 1) == -2 and call(slots=FAKE + 2) == -2 and call(w=FAKE + 1) == -2
    assert call(out=FAKE + 512) == -1                      # inside h
    assert call(base=FAR + 2, out=FAR) == -1               # shifted base
    assert call(tokens=1 << 30, N=8192) == -1


def test_expert_refusals():
    L = qlinear.load()

    def call(path=None, x=FAKE, sx=FAKE, x_rows=64, order=FAKE, div=1, off=FAKE, w=FAKE, sw=FAKE,
             experts=8, y=FAR, scatter=0, slots=64, N=64, K=256, fmt=I8, out=BF16, group=0):
        p = ctypes.byref(path.to_c()) if path else None
        return L.qlin_expert_gemm(p, x, sx, x_rows, order, div, off, w, sw, experts, y, scatter,
                                  slots, N, K, fmt, out, group, None)

    assert call(fmt=BF16) == -1 and call(out=F32) == -1
    assert call(K=200) == -1 and call(N=40) == -1 and call(slots=0) == -1 and call(K=131072) == -1
    assert call(experts=0) == -1 and call(experts=1025) == -1
    assert call(group=64) == -1
    for name in ("x", "sx", "off", "w", "sw", "y"):
        assert call(**{name: None}) == -1
    assert call(div=0) == -1
    assert call(order=None, scatter=1) == -1
    assert call(order=None, x_rows=63) == -1 and call(x_rows=0) == -1
    assert call(x=FAKE + 8) == -2 and call(w=FAKE + 8) == -2 and call(y=FAR + 4) == -2
    assert call(y=FAKE + 64 * 256 - 16) == -1 and b"overlaps" in L.qlin_last_error()
    assert call(sx=FAKE + 2) == -2 and call(sw=FAKE + 4, group=128) == -2
    assert call(order=FAKE + 2) == -2
    assert call(x_rows=1 << 20, K=2048) == -4 and b"2 GiB" in L.qlin_last_error()
    assert call(path=qlinear.Path(qlinear.KIND_SKINNY, 16, 48, 1, 8)) == -4
    good = qlinear.expert_plan(64, 8, 64, 256, I8)
    assert call(path=qlinear.Path(good.kind, good.tokens, good.channels, 2, good.waves)) == -4
    assert call(path=qlinear.Path(good.kind, good.tokens, good.channels, 1, good.waves + 1)) == -4
    wide = qlinear.expert_plan(1 << 16, 8, 4096, 2048, I8)
    assert wide.channels == 256
    assert call(path=wide, group=128) == -4 and b"per-channel" in L.qlin_last_error()
    assert call(slots=1 << 30, order=FAKE, x_rows=1, N=1 << 20, K=16) == -4
    p = qlinear.qlin_path()
    assert L.qlin_expert_plan(64, 8, 64, 256, I8, 0, None) == -1
    assert L.qlin_expert_plan(64, 8, 60, 256, I8, 0, ctypes.byref(p)) == -1


def test_adapter_refusals():
    L = qlinear.load()

    def call(x=FAKE, ldx=256, order=FAKE, off=FAKE, rows=8, n=4, a=FAKE, b=FAKE, rank=16, ranks=None,
             scales=None, base=None, y=FAR, ldy=64, N=64, K=256, t=BF16, ws=None, wsb=0):
        return L.qlin_adapter_add(x, ldx, order, off, rows, n, a, b, rank, ranks, scales, base, y,
                                  ldy, N, K, t, ws, wsb, None)

    assert call(t=F32) == -1 and call(rows=0) == -1 and call(N=40) == -1 and call(K=200) == -1
    assert call(ldx=255) == -1 and call(ldy=63) == -1
    assert call(n=0) == -1 and call(n=1025) == -1
    assert call(rank=0) == -4 and call(rank=129) == -4
    for name in ("x", "order", "off", "a", "b", "y"):
        assert call(**{name: None}) == -1
    assert call(a=FAKE + 8) == -2 and call(b=FAKE + 2) == -2 and call(x=FAKE + 1) == -2
    assert call(order=FAKE + 2) == -2 and call(scales=FAKE + 1) == -2 and call(ranks=FAKE + 2) == -2
    assert call(y=FAKE + 64) == -1 and b"overlaps" in L.qlin_last_error()
    assert call(base=FAR + 2) == -1
    # Column ranges of the same wider rows are apart, or they overlap (rows too many
    # for the call stand for "passed this check").
    wide = dict(ldx=512, ldy=512, rows=1 << 22, ws=FAKE, wsb=1 << 60)
    for apart, status in ((256, -4), (448, -4), (255, -1), (449, -1), (-64, -4), (-63, -1), (0, -1)):
        assert call(y=FAKE + 2 * apart, **wide) == status, apart
    assert call(y=FAKE + 512, **dict(wide, ldy=520)) == -1  # not the same rows
    need = L.qlin_adapter_workspace_bytes(4096, 4, 6144, 64)
    assert need > 0 and L.qlin_adapter_workspace_bytes(1, 4, 6144, 64) == 0
    big = dict(rows=4096, K=6144, ldx=6144, rank=64)
    assert call(**big) == -3 and call(ws=FAKE, wsb=need - 1, **big) == -3
    assert call(ws=FAKE + 4, wsb=need, **big) == -2
    assert call(rows=1 << 22, ws=FAKE, wsb=1 << 60) == -4 and b"2 GiB" in L.qlin_last_error()
    assert call(rows=1 << 25, N=1 << 20, ldy=1 << 20, K=16, ldx=16, x=1 << 60, ws=FAKE, wsb=1 << 60) == -4
    assert b"tiles" in L.qlin_last_error()


def test_binding_refusals():
    """Shapes and types that the Python binding turns away itself."""
    i32 = torch.int32
    order, offsets = torch.zeros(4, dtype=i32), torch.zeros(3, dtype=i32)
    with pytest.raises(ValueError):
        qlinear.group_rows(torch.zeros(4, dtype=torch.int64), 2)
    with pytest.raises(ValueError):
        qlinear.route(torch.zeros(4, 8, dtype=torch.int8), 2)
    with pytest.raises(ValueError):
        qlinear.combine(torch.zeros(4, 8), torch.zeros(2, 2, dtype=i32))
    h = torch.zeros(4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        qlinear.combine(h, torch.zeros(2, 2, dtype=i32), torch.zeros(2, 3))
    with pytest.raises(ValueError):
        qlinear.combine(h, torch.zeros(2, 2, dtype=i32), base=torch.zeros(3, 8, dtype=torch.bfloat16))
    x, w = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(2, 16, 32, dtype=torch.uint8)
    with pytest.raises(ValueError):
        qlinear.expert_gemm(x, torch.zeros(4), w, torch.zeros(2, 15), I8, offsets)
    with pytest.raises(ValueError):
        qlinear.expert_gemm(x, torch.zeros(4), w, torch.zeros(2, 16), I8, offsets[:2])
    with pytest.raises(ValueError):
        qlinear.expert_gemm(x[:, :16], torch.zeros(4), w, torch.zeros(2, 16), I8, offsets)
    xb, a = torch.zeros(4, 32, dtype=torch.bfloat16), torch.zeros(2, 8, 32, dtype=torch.bfloat16)
    b, y = torch.zeros(2, 16, 8, dtype=torch.bfloat16), torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        qlinear.adapter_add(xb, order, offsets, a, b.float(), y)
    with pytest.raises(ValueError):
        qlinear.adapter_add(xb, order[:3], offsets, a, b, y)
    with pytest.raises(ValueError):
        qlinear.adapter_add(xb, order, offsets, a, b, y, base=torch.zeros(4, 32, dtype=torch.bfloat16)[:, :16])


def test_small_adapter_calls_need_no_workspace():
    """The bound below which the binding does not ask: no adapter count or rank needs one there."""
    for rows in (1, 15, 16, 64, 511, 1000, 4096):
        K = ((1 << 17) - 1) // rows // 16 * 16
        for adapters in (1, 2, rows, 1024):
            for rank in (1, 16, 17, 32, 64, 65, 128):
                assert K < 16 or qlinear.adapter_workspace_bytes(rows, adapters, K, rank) == 0
    assert qlinear.adapter_workspace_bytes(64, 64, 2048, 128) > 0


def test_a_workspace_is_dense():
    """Writes of a strided workspace's size would run into what lies between."""
    i32 = torch.int32
    wide = torch.zeros(1 << 16, 2, dtype=torch.uint8)
    ids = torch.zeros(5000, dtype=i32)
    x, sx = torch.zeros(8, 4096, dtype=torch.uint8), torch.zeros(8)
    w, sw = torch.zeros(16, 4096, dtype=torch.uint8), torch.zeros(16)
    path = qlinear.Path(qlinear.KIND_SKINNY, 16, 16, 2, 8)
    assert qlinear.workspace_bytes(path, 8, 16, 4096, I8) > 0
    for call in (lambda ws: qlinear.gemm(x, sx, w, sw, I8, path=path, workspace=ws),
                 lambda ws: qlinear.gemm_finish(x, sx, w, sw, I8, path=path, workspace=ws),
                 lambda ws: qlinear.linear(x.view(torch.bfloat16), w[:, :2048].contiguous(), sw, I8, path=path,
                                           scratch=(x, sx), workspace=ws),
                 lambda ws: qlinear._buffer(ws, 1 << 16, ids.device, None)):
        with pytest.raises(ValueError, match="dense"):
            call(wide[:, 0])


def test_sizes_past_32_bits():
    """Sizes and strides whose low 32 bits would be another, valid call."""
    i32, bf = torch.int32, torch.bfloat16
    meta = lambda *s, dtype=i32: torch.empty(*s, dtype=dtype, device="meta")
    far = (1 << 32) + 8
    u8, f32 = torch.uint8, torch.float32
    calls = [
        lambda: qlinear.group_rows(meta(far), 4),
        lambda: qlinear.group_rows(meta(8), far),
        lambda: qlinear.route(meta(far, 16, dtype=bf), 2),
        lambda: qlinear.route(meta(2, 16, dtype=bf).as_strided((2, 16), (far, 1)), 2),
        lambda: qlinear.route(meta(2, 16, dtype=bf), far),
        lambda: qlinear.combine(meta(far, 16, dtype=bf), meta(4, 2)),
        lambda: qlinear.combine(meta(8, 16, dtype=bf), meta(far, 2)),
        lambda: qlinear.expert_gemm(meta(far, 16, dtype=u8), meta(far, dtype=f32), meta(2, 16, 16, dtype=u8),
                                    meta(2, 16, dtype=f32), I8, meta(3)),
        lambda: qlinear.expert_gemm(meta(8, 16, dtype=u8), meta(8, dtype=f32), meta(2, 16, 16, dtype=u8),
                                    meta(2, 16, dtype=f32), I8, meta(3), order=meta(far)),
        lambda: qlinear.expert_gemm(meta(8, 16, dtype=u8), meta(8, dtype=f32), meta(2, 16, 16, dtype=u8),
                                    meta(2, 16, dtype=f32), I8, meta(3), order=meta(8), divisor=far),
        lambda: qlinear.adapter_add(meta(far, 16, dtype=bf), meta(far), meta(3), meta(2, 8, 16, dtype=bf),
                                    meta(2, 16, 8, dtype=bf), meta(far, 16, dtype=bf)),
        lambda: qlinear.adapter_add(meta(4, 16, dtype=bf), meta(4), meta(3), meta(2, 8, 16, dtype=bf),
                                    meta(2, 16, 8, dtype=bf), meta(4, 16, dtype=bf).as_strided((4, 16), (far, 1))),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(ValueError, match="2.31"):
            call()


OUT = FAR * 20  # of a call's output; the other arrays far from it and from each other


def refuses_overlaps(call, at, size, arrays):
    """Each of `arrays` (argument -> bytes) on the first and on the last 16 bytes of the
    `size` bytes that the call writes at `at`."""
    for name, n in arrays.items():
        for where in (at - (n - 1) // 16 * 16, at + (size - 1) // 16 * 16):
            assert call(**{name: where}) == -1 and b"overlap" in qlinear.load().qlin_last_error(), (name, where)


def test_combine_output_is_apart():
    def call(h=FAR, slots=SLOTS, w=WEIGHTS, base=None):
        return qlinear.load().qlin_combine(h, 8, slots, w, base, OUT, 40, 2, 64, BF16, None)

    refuses_overlaps(call, OUT, 40 * 64 * 2, {"h": 8 * 64 * 2, "slots": 40 * 2 * 4, "w": 40 * 2 * 4})


@pytest.mark.parametrize("group,blocks", [(0, 1), (128, 3)])
def test_expert_output_is_apart(group, blocks):
    rows, slots, experts, N, K = 24, 40, 8, 64, 272

    def call(x=FAR, sx=FAR * 2, order=FAR * 3, off=FAR * 4, w=FAR * 5, sw=FAR * 6):
        return qlinear.load().qlin_expert_gemm(None, x, sx, rows, order, 2, off, w, sw, experts, OUT, 0, slots,
                                               N, K, I8, BF16, group, None)

    refuses_overlaps(call, OUT, slots * N * 2,
                     {"x": rows * K, "sx": blocks * rows * 4, "order": slots * 4, "off": (experts + 1) * 4,
                      "w": experts * N * K, "sw": blocks * experts * N * 4})


def adapter_call(rows, n, rank, N, K, ldy, ws=None, wsb=0):
    def call(x=FAR, order=FAR * 2, off=FAR * 3, a=FAR * 4, b=FAR * 5, ranks=FAR * 6, scales=FAR * 7, base=FAR * 8,
             y=OUT, ws=ws):
        return qlinear.load().qlin_adapter_add(x, K, order, off, rows, n, a, b, rank, ranks, scales, base, y, ldy,
                                               N, K, BF16, ws, wsb, None)
    return call


def test_adapter_output_is_apart():
    rows, n, rank, N, K = 40, 3, 16, 64, 256
    sizes = {"order": rows * 4, "off": (n + 1) * 4, "a": n * rank * K * 2, "b": n * N * rank * 2, "ranks": n * 4,
             "scales": n * 4}
    refuses_overlaps(adapter_call(rows, n, rank, N, K, N), OUT, rows * N * 2, sizes)
    # A column range of wider rows: whatever reaches from the gap into a row, or spans one.
    call = adapter_call(rows, n, rank, N, K, N + 32)
    refuses_overlaps(call, OUT, ((rows - 1) * (N + 32) + N) * 2, sizes)
    for name in ("off", "ranks", "scales"):
        for at in (OUT + N * 2 - 4, OUT + (N + 32) * 2 - 4):
            assert call(**{name: at}) == -1 and b"overlap" in qlinear.load().qlin_last_error(), (name, at)


def test_adapter_workspace_is_apart():
    rows, n, rank, N, K = 4096, 4, 64, 64, 6144
    need = qlinear.adapter_workspace_bytes(rows, n, K, rank)
    assert need > 0
    call = adapter_call(rows, n, rank, N, K, N, FAR * 30, need)
    refuses_overlaps(call, FAR * 30, need,
                     {"order": rows * 4, "off": (n + 1) * 4, "a": n * rank * K * 2, "b": n * N * rank * 2,
                      "ranks": n * 4, "scales": n * 4, "x": rows * K * 2, "base": rows * N * 2, "y": rows * N * 2})


def test_grouping_workspace_is_apart():
    L = qlinear.load()
    count, groups, at = 5000, 40, FAR * 30
    need = L.qlin_group_rows_workspace_bytes(count, groups)

    def rows(ids=IDS, order=ORDER, slots=SLOTS, offsets=OFFSETS):
        return L.qlin_group_rows(ids, count, groups, order, slots, offsets, at, need, None)

    index = {"ids": count * 4, "order": count * 4, "slots": count * 4, "offsets": (groups + 1) * 4}
    refuses_overlaps(rows, at, need, index)

    def route(logits=FAR * 20, ids=IDS, weights=WEIGHTS, order=ORDER, slots=SLOTS, offsets=OFFSETS):
        return L.qlin_route(logits, groups, F32, count // 4, groups, 4, 0, ids, weights, order, slots, offsets, at,
                            need, None)

    refuses_overlaps(route, at, need, {**index, "weights": count * 4, "logits": count // 4 * groups * 4})


def test_grids_past_a_launch():
    """2^32 threads and more are refused before the launch."""
    L = qlinear.load()
    assert L.qlin_combine(FAR, 8, FAR * 2, None, None, OUT, 1 << 24, 1, 8, BF16, None) == -1
    assert b"capacity" in L.qlin_last_error()
    for tokens, experts in (((1 << 28) - 1, 2), ((1 << 26) - 1, 129)):
        need = L.qlin_group_rows_workspace_bytes(tokens, experts)
        assert L.qlin_route(FAR * 20, experts, BF16, tokens, experts, 1, 0, IDS, WEIGHTS, ORDER, SLOTS, OFFSETS,
                            FAR * 30, need, None) == -4
        assert b"capacity" in L.qlin_last_error()
    # 32-token tiles of 64 channels, four waves: 2^24 of them
    assert qlinear.expert_plan(1 << 10, 1 << 9, 1 << 16, 128, I8) == qlinear.Path(qlinear.KIND_TILED, 32, 64, 1, 4)
    rows, N = 1 << 14, 1 << 21
    path = qlinear.Path(qlinear.KIND_TILED, 32, 64, 1, 4)
    assert L.qlin_expert_gemm(ctypes.byref(path.to_c()), FAR, FAR * 2, rows, None, 1, FAR * 3, FAR * 4, FAR * 5, 1,
                              OUT, 0, rows, N, 16, I8, BF16, 0, None) == -4
    assert b"tiles" in L.qlin_last_error()
    rows, N, rank = 1 << 20, 1 << 16, 64
    need = qlinear.adapter_workspace_bytes(rows, 1, 16, rank)
    assert need > 0
    assert L.qlin_adapter_add(FAR, 16, FAR * 2, FAR * 3, rows, 1, FAR * 4, FAR * 5, rank, None, None, None, OUT, N,
                              N, 16, BF16, FAR * 30, need, None) == -4
    assert b"tiles" in L.qlin_last_error()
