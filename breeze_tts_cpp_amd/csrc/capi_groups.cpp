// C ABI of the operators on rows grouped by the weights they use: argument
// checks, tile planning and dispatch. No exceptions cross this boundary.
#include "../../include/qlinear.h"

#include <hip/hip_runtime.h>

#include <climits>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "qlin_internal.hpp"

namespace {

int fail(int status, const char *fmt, ...) {
    char message[512];
    va_list args;
    va_start(args, fmt);
    vsnprintf(message, sizeof(message), fmt, args);
    va_end(args);
    return qlin::set_error(status, message);
}

bool aligned(const void *p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_launch(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(QLIN_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
    return qlin::set_error(QLIN_OK, "");
}

// The byte ranges [a, a + an) and [b, b + bn) share a byte.
bool overlap(const void *a, size_t an, const void *b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}

// So do rows of `an` and `bn` columns, strides lda and ldb (16-bit elements). Column
// ranges of the same wider rows do not.
bool rows_overlap(const void *a, int lda, int an, const void *b, int ldb, int bn, int rows) {
    if (!overlap(a, (size_t(rows - 1) * lda + an) * 2, b, (size_t(rows - 1) * ldb + bn) * 2)) return false;
    if (rows == 1 || lda != ldb) return true;
    const intptr_t apart = (reinterpret_cast<intptr_t>(b) - reinterpret_cast<intptr_t>(a)) / 2;
    const intptr_t column = (apart % lda + lda) % lda;  // of b's first element in a's rows
    return column < an || column + bn > lda;
}

// The rows [a, a + an) of stride lda (16-bit elements) and the bytes [b, b + bn) share one; an
// array that lies between two rows does not.
bool rows_overlap_bytes(const void *a, int lda, int an, int rows, const void *b, size_t bn) {
    if (!b || !overlap(a, (size_t(rows - 1) * lda + an) * 2, b, bn)) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), row = size_t(lda) * 2;
    return y < x || (y - x) % row < size_t(an) * 2 || (y - x) % row + bn > row;
}

// A launch has fewer than 2^32 threads.
bool grid_fits(long workgroups, long threads) { return workgroups <= long(UINT32_MAX) / threads; }

// Most ids of one grouping (index arithmetic past the last run stays in int).
constexpr int kMaxIds = 1 << 30;

int check_grouping(const char *what, const int *ids, long count, int groups, const int *order,
                   const int *slots, const int *offsets, const void *workspace, size_t bytes) {
    if (count < 1 || count > kMaxIds)
        return fail(QLIN_ERR_INVALID, "%s: %ld ids (1 to %d)", what, count, kMaxIds);
    if (groups < 1 || groups > qlin::kMaxGroups)
        return fail(QLIN_ERR_INVALID, "%s: %d groups (1 to %d)", what, groups, qlin::kMaxGroups);
    if (!ids || !order || !slots || !offsets)
        return fail(QLIN_ERR_INVALID, "%s: null pointer", what);
    if (!aligned(ids, 4) || !aligned(order, 4) || !aligned(slots, 4) || !aligned(offsets, 4))
        return fail(QLIN_ERR_ALIGNMENT, "%s: index arrays must be 4-byte aligned", what);
    const size_t flat = size_t(count) * 4;
    const struct { const void *p; size_t bytes; } arrays[] = {
        {ids, flat}, {order, flat}, {slots, flat}, {offsets, size_t(groups + 1) * 4}};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (overlap(arrays[i].p, arrays[i].bytes, arrays[j].p, arrays[j].bytes))
                return fail(QLIN_ERR_INVALID, "%s: ids, order, slots and offsets overlap", what);
    const size_t need = qlin::group_workspace_bytes(int(count), groups);
    if (need && (!workspace || bytes < need))
        return fail(QLIN_ERR_WORKSPACE, "%s: workspace of %zu bytes needed, %zu given", what, need,
                    workspace ? bytes : size_t(0));
    if (need && !aligned(workspace, 4))
        return fail(QLIN_ERR_ALIGNMENT, "%s: workspace must be 4-byte aligned", what);
    // (The placing launch reads the counts there while it writes order and slots.)
    for (const auto &a : arrays)
        if (need && overlap(workspace, need, a.p, a.bytes))
            return fail(QLIN_ERR_INVALID, "%s: workspace overlaps ids, order, slots or offsets", what);
    return QLIN_OK;
}

// The macro tile (index of kExpertTiles) for `slots` rows in `experts` groups,
// of whose sizes the host knows no more than their mean. Measured with uneven
// groups (weights from HBM, 80 shapes of 8-64 experts, 1024-4096 channels, K
// 1024-4096, 0.25-1024 rows per expert, INT8 and FP8):
//  - up to 8 rows per expert the weights' bytes are all: 64x32 tiles, two
//    workgroups per CU (32 experts of 2048 x 2048, 4 rows each: 24.6 us, 26.7 with the
//    K-sliced 32x16 tile). Where they would leave CUs without work, the K-sliced
//    tile has twice the workgroups, each a quarter of the K walk (16 of 1024 x
//    4096, 1 row: 10.1 us against 13.0; 8 of 64, 2048 x 2048: 8.4 against 8.9; with K
//    groups there 11.9 against 10.3, 2 of 8, 4096 x 2048, 7.3 against 9.2), with K above
//    2048 up to 16 rows (16 of 1024 x 4096: 19.4 against 20.8 and 21.3);
//  - up to 31 rows 128x64 (16 rows: 27.6 us against 29.8 on 64x32, 27.9 on 128x128),
//    but 64x32 up to 32 rows where 128-channel tiles leave CUs without work (16 of
//    1024 x 4096, 16 rows: 20.9 against 23.5), where also up to 96 rows 128x64 gives
//    more of them some (64 rows: 24.6 against 26.9 on 128x128);
//  - up to 127 rows 128x128 (64 rows: 36.7 us, 37.0 on 128x64, 48.6 on 256x256);
//  - above, of 128x128 (two workgroups per CU) and 256x256 the tile whose rounds of
//    workgroups cost least, at the time that a round of each takes with uneven
//    groups, a part per 128 of K and a fixed one (prologue, epilogue).
// With K groups 128x64 from 4 rows (6 rows, 31 experts of 2064 x 2048: 23.5 us, 26.7 on
// 64x32), at any size: beside the scales' registers a 128x128 tile is level (125 rows, 64
// experts of 2048 x 1024: 54-59 us in five forms against 56). Many rows pay for it (512 rows
// each, 32 experts of 4096 x 2048: INT8 304 us, FP8 282, per channel 174 and 167).
// On the 80 shapes the choice is within 5% of the best tile, with K groups on as many
// within 10%. Groups far from the mean cost more: 4000 rows that all fall to one of 512
// experts, 1024 x 1024 INT8, 28.8 us (22.1 on 256x256), of 64 experts within 11%.
int choose_tile(long slots, int experts, int N, int K, int group) {
    const long each = slots / experts;
    const long some = slots < experts ? slots : experts;  // groups that can have rows
    const bool few = some * ((N + 63) / 64) <= (group && K <= 2048 ? 128 : 256);
    if (few && each <= (!group && K > 2048 ? 16 : 8)) return 0;
    if (each <= (group ? 3 : 8)) return 1;
    const bool idle = some * ((N + 127) / 128) < 256;  // CUs
    if (each <= 32 && idle) return 1;
    if (group || each < 32 || (each <= 96 && idle)) return 2;
    if (each < 128) return 3;
    constexpr struct { int tile; long per_round; double stage, fixed; } kCost[] = {
        {3, 512, 900, 6000}, {4, 256, 1350, 9000}};  // ns
    const double stages = double((long(K) + 127) / 128);
    int best = 3;
    double least = 1e300;
    for (const auto &c : kCost) {
        const auto &t = qlin::kExpertTiles[c.tile];
        // A group's last tile is short: on average 0.6 of a tile more, at least one.
        const long rows = slots / t.tokens + experts * 3L / 5;
        const long tiles = (rows > experts ? rows : experts) * ((N + t.channels - 1) / t.channels);
        // Whole rounds while they are few; many even out to half a round more.
        const long rounds2 = tiles <= 4 * c.per_round ? (tiles + c.per_round - 1) / c.per_round * 2
                                                      : tiles * 2 / c.per_round + 1;
        const double cost = double(rounds2) * (stages * c.stage + c.fixed);
        if (cost < least) least = cost, best = c.tile;
    }
    return best;
}

int tile_index(const qlin_path &p) {
    int i = 0;
    for (const auto &t : qlin::kExpertTiles) {
        if (t.channels == p.channels && t.tokens == p.tokens && t.waves == p.waves &&
            (p.kind == QLIN_KIND_SKINNY) == (t.slices > 1))
            return i;
        ++i;
    }
    return -1;
}

int check_expert_shape(int slots, int experts, int N, int K, int fmt, int group) {
    if (fmt != QLIN_I8 && fmt != QLIN_FP8)
        return fail(QLIN_ERR_INVALID, "unsupported quantized storage type");
    if (slots < 1 || slots > kMaxIds || N < 1 || K < 1 || K % 16 || N % 16)
        return fail(QLIN_ERR_INVALID, "grouped GEMM unsupported shape slots=%d N=%d K=%d", slots, N, K);
    if (experts < 1 || experts > qlin::kMaxGroups)
        return fail(QLIN_ERR_INVALID, "grouped GEMM: %d experts (1 to %d)", experts, qlin::kMaxGroups);
    if (fmt == QLIN_I8 && K > INT32_MAX / (128 * 128))
        return fail(QLIN_ERR_INVALID, "INT8 reduction can overflow INT32");
    if (group != 0 && group != 128)
        return fail(QLIN_ERR_INVALID, "grouped GEMM scales are per channel (0) or per 128 of K (got %d)",
                    group);
    return QLIN_OK;
}

}  // namespace

extern "C" {

size_t qlin_group_rows_workspace_bytes(int count, int groups) {
    if (count < 1 || count > kMaxIds || groups < 1 || groups > qlin::kMaxGroups) return 0;
    return qlin::group_workspace_bytes(count, groups);
}

int qlin_group_rows(const int *ids, int count, int groups, int *order, int *slots, int *offsets,
                    void *workspace, size_t workspace_bytes, qlin_stream_t stream) {
    const int status = check_grouping("group_rows", ids, count, groups, order, slots, offsets,
                                      workspace, workspace_bytes);
    if (status) return status;
    qlin::launch_group_rows({ids, count, groups, order, slots, offsets, workspace},
                            reinterpret_cast<hipStream_t>(stream));
    return check_launch("group_rows launch");
}

int qlin_route(const void *logits, int ld, int logits_type, int tokens, int experts, int top_k,
               int normalize, int *ids, float *weights, int *order, int *slots, int *offsets,
               void *workspace, size_t workspace_bytes, qlin_stream_t stream) {
    if (logits_type != QLIN_F32 && logits_type != QLIN_BF16 && logits_type != QLIN_F16)
        return fail(QLIN_ERR_INVALID, "router logits must be F32, BF16 or F16");
    if (tokens < 1 || experts < 1 || experts > qlin::kMaxGroups || ld < experts)
        return fail(QLIN_ERR_INVALID, "router shape tokens=%d experts=%d ld=%d (1 to %d experts)",
                    tokens, experts, ld, qlin::kMaxGroups);
    if (top_k < 1 || top_k > qlin::kMaxTopK || top_k > experts)
        return fail(QLIN_ERR_INVALID, "router top_k=%d of %d experts (1 to %d)", top_k, experts,
                    qlin::kMaxTopK);
    if (!logits || !weights) return fail(QLIN_ERR_INVALID, "router: null pointer");
    if (!aligned(logits, logits_type == QLIN_F32 ? 4 : 2) || !aligned(weights, 4))
        return fail(QLIN_ERR_ALIGNMENT, "router logits and weights must be aligned to their type");
    const int status = check_grouping("router", ids, long(tokens) * top_k, experts, order, slots,
                                      offsets, workspace, workspace_bytes);
    if (status) return status;
    const long each = 256 / (experts <= 128 ? 16 : 64);  // tokens a workgroup
    if (!grid_fits((tokens + each - 1) / each, 256))
        return fail(QLIN_ERR_UNSUPPORTED, "router grid exceeds capacity");
    const size_t logits_bytes = (size_t(tokens - 1) * ld + experts) * (logits_type == QLIN_F32 ? 4 : 2);
    const size_t flat = size_t(tokens) * top_k * 4, index_bytes[] = {flat, flat, flat, size_t(experts + 1) * 4};
    const void *index[] = {ids, order, slots, offsets};
    for (int i = 0; i < 4; ++i)
        if (overlap(index[i], index_bytes[i], logits, logits_bytes) ||
            overlap(index[i], index_bytes[i], weights, flat))
            return fail(QLIN_ERR_INVALID, "router outputs overlap its logits or each other");
    if (overlap(weights, flat, logits, logits_bytes))
        return fail(QLIN_ERR_INVALID, "router outputs overlap its logits or each other");
    const size_t need = qlin::group_workspace_bytes(tokens * top_k, experts);
    if (need && (overlap(workspace, need, logits, logits_bytes) || overlap(workspace, need, weights, flat)))
        return fail(QLIN_ERR_INVALID, "router workspace overlaps its logits or weights");
    qlin::launch_route({logits, ld, logits_type, tokens, experts, top_k, normalize != 0, ids, weights},
                       {ids, tokens * top_k, experts, order, slots, offsets, workspace},
                       reinterpret_cast<hipStream_t>(stream));
    return check_launch("router launch");
}

int qlin_combine(const void *h, int h_rows, const int *slots, const float *weights,
                 const void *base, void *out, int tokens, int top_k, int N, int type,
                 qlin_stream_t stream) {
    if (type != QLIN_BF16 && type != QLIN_F16)
        return fail(QLIN_ERR_INVALID, "combine type must be BF16 or F16");
    if (h_rows < 1 || tokens < 1 || top_k < 1 || top_k > qlin::kMaxTopK || N < 1)
        return fail(QLIN_ERR_INVALID, "combine shape h_rows=%d tokens=%d top_k=%d N=%d", h_rows,
                    tokens, top_k, N);
    if (!grid_fits(long(tokens) * ((long(N) + 2047) / 2048), 256))
        return fail(QLIN_ERR_INVALID, "combine grid exceeds capacity");
    if (!h || !slots || !out) return fail(QLIN_ERR_INVALID, "combine: null pointer");
    if (!aligned(h, 2) || !aligned(base, 2) || !aligned(out, 2) || !aligned(slots, 4) ||
        !aligned(weights, 4))
        return fail(QLIN_ERR_ALIGNMENT, "combine operands must be aligned to their type");
    if (overlap(h, size_t(h_rows) * N * 2, out, size_t(tokens) * N * 2))
        return fail(QLIN_ERR_INVALID, "combine output overlaps its input rows");
    if (base && base != out && overlap(base, size_t(tokens) * N * 2, out, size_t(tokens) * N * 2))
        return fail(QLIN_ERR_INVALID, "combine output overlaps part of its base");
    const size_t choices = size_t(tokens) * top_k * 4;
    if (overlap(slots, choices, out, size_t(tokens) * N * 2) ||
        (weights && overlap(weights, choices, out, size_t(tokens) * N * 2)))
        return fail(QLIN_ERR_INVALID, "combine output overlaps its slots or weights");
    qlin::launch_combine({h, slots, weights, base, out, h_rows, tokens, top_k, N, type},
                         reinterpret_cast<hipStream_t>(stream));
    return check_launch("combine launch");
}

int qlin_expert_plan(int slots, int experts, int N, int K, int fmt, int group, qlin_path *path) {
    if (!path) return fail(QLIN_ERR_INVALID, "path is null");
    const int status = check_expert_shape(slots, experts, N, K, fmt, group);
    if (status) return status;
    const auto &t = qlin::kExpertTiles[choose_tile(slots, experts, N, K, group)];
    *path = {t.slices > 1 ? QLIN_KIND_SKINNY : QLIN_KIND_TILED, t.tokens, t.channels, 1, t.waves, 0};
    return qlin::set_error(QLIN_OK, "");
}

int qlin_expert_gemm(const qlin_path *path, const void *x, const float *sx, int x_rows,
                     const int *order, int divisor, const int *offsets, const void *w,
                     const float *sw, int experts, void *y, int scatter, int slots, int N, int K,
                     int fmt, int out_type, int group, qlin_stream_t stream) {
    int status = check_expert_shape(slots, experts, N, K, fmt, group);
    if (status) return status;
    if (out_type != QLIN_BF16 && out_type != QLIN_F16)
        return fail(QLIN_ERR_INVALID, "grouped GEMM output must be F16 or BF16");
    if (!x || !sx || !offsets || !w || !sw || !y)
        return fail(QLIN_ERR_INVALID, "grouped GEMM operand pointer is null");
    if (divisor < 1) return fail(QLIN_ERR_INVALID, "grouped GEMM divisor must be at least 1");
    if (scatter && !order) return fail(QLIN_ERR_INVALID, "scattered results need the rows' order");
    if (x_rows < 1 || (!order && x_rows < slots))
        return fail(QLIN_ERR_INVALID, "grouped GEMM: %d input rows for %d slots", x_rows, slots);
    if (!aligned(x, 16) || !aligned(w, 16))
        return fail(QLIN_ERR_ALIGNMENT, "quantized operands must be 16-byte aligned");
    if (!aligned(y, 8)) return fail(QLIN_ERR_ALIGNMENT, "output must be 8-byte aligned");
    if (!aligned(sx, 4) || !aligned(sw, group ? 16 : 4))
        return fail(QLIN_ERR_ALIGNMENT, "scales must be 4-byte aligned (group weight scales 16-byte)");
    if (!aligned(offsets, 4) || !aligned(order, 4))
        return fail(QLIN_ERR_ALIGNMENT, "index arrays must be 4-byte aligned");
    if (overlap(x, size_t(x_rows) * K, y, size_t(slots) * N * 2))
        return fail(QLIN_ERR_INVALID, "grouped GEMM output overlaps its input");
    // Gathered rows are addressed through one 32-bit buffer range, and so are a
    // tile's rows of either operand.
    if (order && long(x_rows) * K > INT32_MAX)
        return fail(QLIN_ERR_UNSUPPORTED, "gathered input rows exceed 2 GiB");
    // So are the K groups' scales, the tokens' and one expert's.
    if (group && (long(K) + 127) / 128 * (N > x_rows ? N : x_rows) * 4 > INT32_MAX)
        return fail(QLIN_ERR_UNSUPPORTED, "K-group scale arrays exceed 2 GiB");
    int tile = choose_tile(slots, experts, N, K, group);
    if (path && path->kind) {
        tile = path->splits == 1 && path->staged == 0 ? tile_index(*path) : -1;
        if (tile < 0)
            return fail(QLIN_ERR_UNSUPPORTED, "no grouped %dx%d path of %d waves (kind %d)",
                        path->channels, path->tokens, path->waves, path->kind);
        if (group && tile >= qlin::kExpertNarrowTiles)
            return fail(QLIN_ERR_UNSUPPORTED, "grouped %dx%d path has per-channel scales only",
                        path->channels, path->tokens);
    }
    const auto &t = qlin::kExpertTiles[tile];
    if (long(t.channels > t.tokens ? t.channels : t.tokens) * K > INT32_MAX)
        return fail(QLIN_ERR_UNSUPPORTED, "grouped GEMM tile rows exceed 2 GiB");
    if (!grid_fits(qlin::expert_row_tiles(slots, experts, t.tokens) * ((long(N) + t.channels - 1) / t.channels),
                   64 * t.waves))
        return fail(QLIN_ERR_UNSUPPORTED, "grouped GEMM has too many macro tiles for a launch");
    const size_t y_bytes = size_t(slots) * N * 2, blocks = group ? (size_t(K) + 127) / 128 : 1;
    if (overlap(sx, blocks * x_rows * 4, y, y_bytes) || overlap(w, size_t(experts) * N * K, y, y_bytes) ||
        overlap(sw, blocks * experts * N * 4, y, y_bytes) || overlap(offsets, size_t(experts + 1) * 4, y, y_bytes) ||
        (order && overlap(order, size_t(slots) * 4, y, y_bytes)))
        return fail(QLIN_ERR_INVALID, "grouped GEMM output overlaps its weights, scales or indices");
    qlin::ExpertArgs a{static_cast<const uint8_t *>(x), sx, order, offsets,
                       static_cast<const uint8_t *>(w), sw, y, x_rows, divisor, scatter != 0,
                       experts, slots, N, K, fmt, out_type, group};
    const int r = qlin::launch_expert(a, tile, reinterpret_cast<hipStream_t>(stream));
    if (r) return fail(r, "no kernel variant for this path");
    return check_launch("grouped GEMM launch");
}

size_t qlin_adapter_workspace_bytes(int rows, int adapters, int K, int rank) {
    if (rows < 1 || rows > kMaxIds || adapters < 1 || K < 1 || rank < 1) return 0;
    return qlin::adapter_workspace_bytes(rows, adapters, K, rank);
}

int qlin_adapter_add(const void *x, int ldx, const int *order, const int *offsets, int rows,
                     int adapters, const void *a, const void *b, int rank, const int *ranks,
                     const float *scales, const void *base, void *y, int ldy, int N, int K, int type,
                     void *workspace, size_t workspace_bytes, qlin_stream_t stream) {
    if (type != QLIN_BF16 && type != QLIN_F16)
        return fail(QLIN_ERR_INVALID, "adapter type must be BF16 or F16");
    if (rows < 1 || rows > kMaxIds || N < 1 || K < 1 || K % 16 || N % 16 || ldx < K || ldy < N)
        return fail(QLIN_ERR_INVALID, "adapter shape rows=%d N=%d K=%d ldx=%d ldy=%d", rows, N, K,
                    ldx, ldy);
    if (adapters < 1 || adapters > qlin::kMaxGroups)
        return fail(QLIN_ERR_INVALID, "%d adapters (1 to %d)", adapters, qlin::kMaxGroups);
    if (rank < 1 || rank > 128)
        return fail(QLIN_ERR_UNSUPPORTED, "adapter rank %d (1 to 128)", rank);
    if (!x || !order || !offsets || !a || !b || !y)
        return fail(QLIN_ERR_INVALID, "adapter operand pointer is null");
    if (!aligned(a, 16) || !aligned(b, 16))
        return fail(QLIN_ERR_ALIGNMENT, "adapter matrices must be 16-byte aligned");
    if (!aligned(x, 2) || !aligned(base, 2) || !aligned(y, 2))
        return fail(QLIN_ERR_ALIGNMENT, "16-bit rows must be 2-byte aligned");
    if (!aligned(order, 4) || !aligned(offsets, 4) || !aligned(ranks, 4) || !aligned(scales, 4))
        return fail(QLIN_ERR_ALIGNMENT, "index arrays and scales must be 4-byte aligned");
    const size_t x_bytes = (size_t(rows - 1) * ldx + K) * 2;
    if (rows_overlap(x, ldx, K, y, ldy, N, rows))
        return fail(QLIN_ERR_INVALID, "adapter output overlaps its input");
    if (base && base != y && rows_overlap(base, ldy, N, y, ldy, N, rows))
        return fail(QLIN_ERR_INVALID, "adapter output overlaps part of its base");
    const size_t need = qlin::adapter_workspace_bytes(rows, adapters, K, rank);
    if (need && (!workspace || workspace_bytes < need))
        return fail(QLIN_ERR_WORKSPACE, "adapter workspace of %zu bytes needed, %zu given", need,
                    workspace ? workspace_bytes : size_t(0));
    if (need && !aligned(workspace, 16))
        return fail(QLIN_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    // Rows of x and an adapter's a are addressed through 32-bit buffer ranges.
    if (x_bytes > size_t(INT32_MAX) || size_t(rank) * K * 2 > size_t(INT32_MAX))
        return fail(QLIN_ERR_UNSUPPORTED, "adapter input rows exceed 2 GiB");
    // (The second of two launches, up to rank 64: 32 rows and 256 channels a workgroup. Other
    // forms take more channels where the rows are many.)
    if (need && rank <= 64 && !grid_fits(qlin::expert_row_tiles(rows, adapters, 32) * ((long(N) + 255) / 256), 512))
        return fail(QLIN_ERR_UNSUPPORTED, "adapter call has too many tiles for a launch");
    const struct { const void *p; size_t bytes; } inputs[] = {
        {a, size_t(adapters) * rank * K * 2}, {b, size_t(adapters) * N * rank * 2},
        {order, size_t(rows) * 4}, {offsets, size_t(adapters + 1) * 4},
        {ranks, size_t(adapters) * 4}, {scales, size_t(adapters) * 4}};
    for (const auto &in : inputs) {
        if (rows_overlap_bytes(y, ldy, N, rows, in.p, in.bytes))
            return fail(QLIN_ERR_INVALID, "adapter output overlaps its matrices or index arrays");
        if (need && in.p && overlap(workspace, need, in.p, in.bytes))
            return fail(QLIN_ERR_INVALID, "adapter workspace overlaps its matrices or index arrays");
    }
    if (need && (rows_overlap_bytes(y, ldy, N, rows, workspace, need) ||
                 rows_overlap_bytes(x, ldx, K, rows, workspace, need) ||
                 (base && rows_overlap_bytes(base, ldy, N, rows, workspace, need))))
        return fail(QLIN_ERR_INVALID, "adapter workspace overlaps its rows");
    qlin::launch_adapter({x, order, offsets, a, b, ranks, scales, base, y, ldx, ldy, rows, adapters,
                          rank, N, K, type, workspace},
                         reinterpret_cast<hipStream_t>(stream));
    return check_launch("adapter launch");
}

}  // extern "C"
