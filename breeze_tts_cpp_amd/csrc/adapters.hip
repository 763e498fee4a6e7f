// Low-rank adapters of many requests beside a shared projection, for gfx950
// (qlin_adapter_add): for the rows m of adapter g,
//   t[m, r] = sum_k x[m, k] A[g, r, k]                    (r < ranks[g])
//   y[m, n] = s16(base[m, n] + scale[g] * sum_r t[m, r] B[g, n, r])
// with both products on 16-bit MFMAs accumulating in fp32. t stays fp32 until it
// is the second product's operand: there it is two 16-bit numbers, t = hi + lo
// with lo the rounding error of hi (18 bits of t for bf16, 22 for f16, whose
// rows are first scaled by a power of two into f16's range), so t costs one more
// MFMA and no accuracy that the 16-bit result could show.
//
// MFMA operands (v_mfma_f32_16x16x32): the A operand is 16 ranks (then 16
// channels), the B operand 16 tokens, eight consecutive K values per lane, so
// fragments are 16-byte loads straight from global memory; nothing is read
// twice by a workgroup. A lane's result is four consecutive A rows of one token.
#include "qlin_internal.hpp"
#include "row_encode.hpp"
#include "row_groups.hpp"

#include <algorithm>
#include <type_traits>

namespace qlin {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <class T> __device__ __forceinline__ void mma16(f32x4 &c, const uint4 &a, const uint4 &b) {
    if constexpr (std::is_same_v<T, f16_t>)
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                   __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                    __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight 16-bit values p[0 .. 8), zeros from `have` on (p[0] is readable).
template <bool Vec> __device__ __forceinline__ uint4 load_piece(const uint16_t *p, int have) {
    if constexpr (Vec) {
        uint4 v = *reinterpret_cast<const uint4 *>(p);
        if (have < 8) {
            auto keep = [&](uint32_t u, int i) {
                return have > i + 1 ? u : have > i ? u & 0xffffu : 0u;
            };
            v = uint4{keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6)};
        }
        return v;
    } else {
        uint32_t e[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < have ? p[i] : 0;
        return uint4{e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16),
                     e[6] | (e[7] << 16)};
    }
}

// The tile's row ml: its row of x and y, or -1.
__device__ __forceinline__ int source_row(const AdapterArgs &p, const RowTile &t, int ml) {
    if (ml >= t.rows) return -1;
    const int row = p.order[t.begin + ml];
    return uint32_t(row) < uint32_t(p.rows) ? row : -1;
}
__device__ __forceinline__ int group_rank(const AdapterArgs &p, int g) {
    return p.ranks ? min(max(p.ranks[g], 0), p.rank) : p.rank;
}

// acc[i][t] += A rows [16i, 16i + 16) x the tile's tokens [16t, 16t + 16) over the K
// range [k0, k1) (32 at a time; k0 a multiple of 32).
template <class T, int RT, int MT, bool Vec>
__device__ __forceinline__ void shrink(const AdapterArgs &p, const RowTile &tile, int rank, int k0,
                                       int k1, f32x4 (&acc)[RT][MT]) {
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
    const uint16_t *xrow[MT], *arow[RT];
    bool xin[MT], ain[RT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = source_row(p, tile, t * 16 + row16);
        xin[t] = row >= 0;
        xrow[t] = static_cast<const uint16_t *>(p.x) + size_t(max(row, 0)) * p.ldx + quad * 8;
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = i * 16 + row16;
        ain[i] = r < rank;
        arow[i] = static_cast<const uint16_t *>(p.a) +
                  (size_t(tile.group) * p.rank + min(r, p.rank - 1)) * p.K + quad * 8;
    }
    // kDeep steps' loads are issued together, then their products.
    constexpr int kDeep = RT * MT >= 16 ? 1 : RT + MT >= 6 ? 2 : 4;
    for (int k = k0; k < k1; k += 32 * kDeep) {
        uint4 xv[kDeep][MT], av[kDeep][RT];
#pragma unroll
        for (int d = 0; d < kDeep; ++d) {
            const bool in = k + d * 32 + quad * 8 < k1;
            const int at = in ? k + d * 32 : -quad * 8;  // (past the range: the row's start)
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const uint4 v = load_piece<Vec>(xrow[t] + at, 8);
                xv[d][t] = in && xin[t] ? v : uint4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const uint4 v = load_piece<true>(arow[i] + at, 8);
                av[d][i] = in && ain[i] ? v : uint4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int d = 0; d < kDeep; ++d)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) mma16<T>(acc[i][t], av[d][i], xv[d][t]);
    }
}

// One lane of the 16 that share a token: its RP / 16 values of t (ranks l,
// l + 16, ...) into hi and lo [RP] in LDS, and (lane 0) the exponent of the
// token's power-of-two scale.
template <class T, int RP>
__device__ __forceinline__ void split_token(const float (&t)[RP / 16], uint16_t *hi, uint16_t *lo,
                                            int *exponent) {
    const int l = threadIdx.x & 15;
    int e = 0;
    if constexpr (std::is_same_v<T, f16_t>) {
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < RP / 16; ++i) {
            const float v = fabsf(t[i]);
            most = fmaxf(most, v < __builtin_inff() ? v : 0.f);
        }
        most = group_max<16>(most);
        // 2^e <= most < 2^(e + 1); scaled below 2^15.
        e = most > 0.f ? __builtin_amdgcn_frexp_expf(most) - 1 - 14 : 0;
    }
#pragma unroll
    for (int i = 0; i < RP / 16; ++i) {
        const float v = __builtin_amdgcn_ldexpf(t[i], -e);
        const uint16_t h = from_float(v, T{});
        const float back = to_float(h, T{});
        const float rest = v - back;
        hi[l + 16 * i] = h;
        lo[l + 16 * i] = fabsf(back) < __builtin_inff() ? from_float(rest, T{}) : uint16_t(0);
    }
    if (l == 0) *exponent = e;
}

// The second product for channels [n0, n0 + 32) and the tile's tokens, added to
// base and stored. hi / lo: [16 MT][RP + 8] in LDS. MFMA row p of fragment f
// is channel 8 (p / 4) + 4 f + p % 4 of the 32, so a lane's two fragments are
// eight consecutive channels.
template <class T, int RP, int MT, bool VecB, bool VecY>
__device__ __forceinline__ void expand(const AdapterArgs &p, const RowTile &tile, int rank, int n0,
                                       const uint16_t *hi, const uint16_t *lo, const int *exponent,
                                       float scale) {
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
    constexpr int kSteps = RP / 32, kPitch = RP + 8;
    uint4 bv[2][kSteps];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        const int n = n0 + 8 * (row16 / 4) + 4 * f + row16 % 4;
        const uint16_t *row = static_cast<const uint16_t *>(p.b) +
                              (size_t(tile.group) * p.N + min(n, p.N - 1)) * p.rank;
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int r = s * 32 + quad * 8;
            const int have = n < p.N ? min(rank - r, 8) : 0;
            bv[f][s] = have > 0 ? load_piece<VecB>(row + r, have) : uint4{0, 0, 0, 0};
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int ml = t * 16 + row16, row = source_row(p, tile, ml), n = n0 + quad * 8;
        const bool live = row >= 0 && n < p.N;
        const size_t at = size_t(max(row, 0)) * p.ldy + n;
        float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (live && p.base)
            load8<T, VecY>(static_cast<const uint16_t *>(p.base) + at, 0, 8, v);
        f32x4 acc[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const uint4 h = *reinterpret_cast<const uint4 *>(hi + ml * kPitch + s * 32 + quad * 8);
            const uint4 l = *reinterpret_cast<const uint4 *>(lo + ml * kPitch + s * 32 + quad * 8);
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                mma16<T>(acc[f], bv[f][s], l);
                mma16<T>(acc[f], bv[f][s], h);
            }
        }
        const int e = exponent[ml];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] += scale * __builtin_amdgcn_ldexpf(acc[i / 4][i % 4], e);
        if (live) store16x8<T, VecY>(static_cast<uint16_t *>(p.y) + at, 0, 8, v);
    }
}

// t of a tile from the waves' partial sums in LDS ([parts][16 MT][RP]; they
// may be the workspace's, part_stride floats apart) to hi / lo.
template <class T, int RP, int MT>
__device__ __forceinline__ void gather_t(const float *parts, int count, size_t part_stride,
                                         int live_rows, int rank, uint16_t *hi, uint16_t *lo,
                                         int *exponent) {
    for (int ml = threadIdx.x / 16; ml < 16 * MT; ml += blockDim.x / 16) {
        float t[RP / 16];
#pragma unroll
        for (int i = 0; i < RP / 16; ++i) t[i] = 0.f;
        if (ml < live_rows)
            for (int q = 0; q < count; ++q)
#pragma unroll
                for (int i = 0; i < RP / 16; ++i)
                    t[i] += parts[q * part_stride + size_t(ml) * RP + i * 16 + threadIdx.x % 16];
        // (Past the rank A was read as zeros, but 0 * inf is NaN.)
#pragma unroll
        for (int i = 0; i < RP / 16; ++i)
            if (i * 16 + int(threadIdx.x % 16) >= rank) t[i] = 0.f;
        split_token<T, RP>(t, hi + ml * (RP + 8), lo + ml * (RP + 8), exponent + ml);
    }
}

constexpr int rank_pad(int rt) { return rt < 2 ? 32 : 16 * rt; }

// ---------------------------------------------------------------- one launch
// A 16-row tile's whole work in one workgroup: its eight waves split K of the
// first product, sum through LDS, and split the tile's channels of the second.
// Every column tile of the same rows repeats the first product.
template <class T, int RT, bool VecX, bool VecB, bool VecY>
__global__ __launch_bounds__(512) void adapter_one(AdapterArgs p, int columns, int width) {
    constexpr int RP = rank_pad(RT), W = 8;
    __shared__ __attribute__((aligned(16))) float parts[W * 16 * RP];
    __shared__ __attribute__((aligned(16))) uint16_t hi[16 * (RP + 8)], lo[16 * (RP + 8)];
    __shared__ int exponent[16];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16, columns, blockIdx.x, tile)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row16 = lane & 15, quad = lane >> 4;
    const int rank = group_rank(p, tile.group);
    const float scale = p.scales ? p.scales[tile.group] : 1.f;
    f32x4 acc[RT][1];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i][0] = f32x4{0, 0, 0, 0};
    const int span = ((p.K + 31) / 32 + W - 1) / W * 32;
    shrink<T, RT, 1, VecX>(p, tile, rank, min(wave * span, p.K), min((wave + 1) * span, p.K), acc);
#pragma unroll
    for (int i = 0; i < RP / 16; ++i)
        *reinterpret_cast<f32x4 *>(parts + (wave * 16 + row16) * RP + i * 16 + quad * 4) =
            i < RT ? acc[i < RT ? i : 0][0] : f32x4{0, 0, 0, 0};
    __syncthreads();
    gather_t<T, RP, 1>(parts, W, 16 * RP, 16, rank, hi, lo, exponent);
    __syncthreads();
    const int n_end = min((tile.column + 1) * width, p.N);
    for (int n0 = tile.column * width + wave * 32; n0 < n_end; n0 += W * 32)
        expand<T, RP, 1, VecB, VecY>(p, tile, rank, n0, hi, lo, exponent, scale);
}

// ---------------------------------------------------------------- two launches
// First product: a 64-row tile's K range split over the grid and four waves;
// partial t [split][slot][RP] to the workspace.
template <class T, int RT, bool VecX>
__global__ __launch_bounds__(256) void adapter_shrink(AdapterArgs p, int splits) {
    constexpr int RP = rank_pad(RT), W = 4, MT = 4;
    __shared__ __attribute__((aligned(16))) float parts[W * 16 * RP];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16 * MT, splits, blockIdx.x, tile)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row16 = lane & 15, quad = lane >> 4;
    const int rank = group_rank(p, tile.group);
    f32x4 acc[RT][MT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int ranges = W * splits, span = ((p.K + 31) / 32 + ranges - 1) / ranges * 32;
    const int k0 = min((tile.column * W + wave) * span, p.K);
    shrink<T, RT, MT, VecX>(p, tile, rank, k0, min(k0 + span, p.K), acc);
    float *out = static_cast<float *>(p.workspace) +
                 (size_t(tile.column) * p.rows + tile.begin) * RP;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < RP / 16; ++i)
            *reinterpret_cast<f32x4 *>(parts + (wave * 16 + row16) * RP + i * 16 + quad * 4) =
                i < RT ? acc[i < RT ? i : 0][t] : f32x4{0, 0, 0, 0};
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * RP; i += 256) {
            if (t * 16 + i / RP >= tile.rows) break;
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < W; ++q) s += parts[q * 16 * RP + i];
            out[size_t(t) * 16 * RP + i] = s;
        }
    }
}

template <class T, int RT, bool VecB, bool VecY>
__global__ __launch_bounds__(256) void adapter_expand(AdapterArgs p, int splits, int columns,
                                                      int width) {
    constexpr int RP = rank_pad(RT), MT = 4, W = 4;
    __shared__ __attribute__((aligned(16))) uint16_t hi[64 * (RP + 8)], lo[64 * (RP + 8)];
    __shared__ int exponent[64];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16 * MT, columns, blockIdx.x, tile)) return;
    const int wave = threadIdx.x >> 6;
    const int rank = group_rank(p, tile.group);
    const float scale = p.scales ? p.scales[tile.group] : 1.f;
    gather_t<T, RP, MT>(static_cast<const float *>(p.workspace) + size_t(tile.begin) * RP, splits,
                        size_t(p.rows) * RP, tile.rows, rank, hi, lo, exponent);
    __syncthreads();
    const int n_end = min((tile.column + 1) * width, p.N);
    for (int n0 = tile.column * width + wave * 32; n0 < n_end; n0 += W * 32)
        expand<T, RP, MT, VecB, VecY>(p, tile, rank, n0, hi, lo, exponent, scale);
}

struct AdapterPlan {
    bool one;
    int splits, columns, width;
};
AdapterPlan plan_adapter(int rows, int adapters, int N, int K, int rank) {
    (void)rank;
    AdapterPlan p{};
    p.one = rows <= 64;
    const long tiles = expert_row_tiles(rows, adapters, p.one ? 16 : 64);
    const long wanted = std::max(1L, (p.one ? 256 : 512) / tiles);
    const int unit = p.one ? 256 : 128;
    p.columns = int(std::min(wanted, long(N + unit - 1) / unit));
    p.width = ((N + unit - 1) / unit + p.columns - 1) / p.columns * unit;
    p.columns = (N + p.width - 1) / p.width;
    p.splits = p.one ? 0 : int(std::min(std::min(wanted, 8L), long(K + 255) / 256));
    return p;
}

template <class T, int RT, bool VecX, bool VecB, bool VecY>
void launch_as(const AdapterArgs &a, const AdapterPlan &p, hipStream_t s) {
    const int tiles = int(expert_row_tiles(a.rows, a.adapters, p.one ? 16 : 64));
    if (p.one) {
        hipLaunchKernelGGL((adapter_one<T, RT, VecX, VecB, VecY>), dim3(unsigned(tiles * p.columns)),
                           dim3(512), 0, s, a, p.columns, p.width);
        return;
    }
    hipLaunchKernelGGL((adapter_shrink<T, RT, VecX>), dim3(unsigned(tiles * p.splits)), dim3(256), 0,
                       s, a, p.splits);
    hipLaunchKernelGGL((adapter_expand<T, RT, VecB, VecY>), dim3(unsigned(tiles * p.columns)),
                       dim3(256), 0, s, a, p.splits, p.columns, p.width);
}

template <class T, int RT>
void launch_rank(const AdapterArgs &a, const AdapterPlan &p, hipStream_t s) {
    auto at16 = [](const void *q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
    const bool x = a.ldx % 8 == 0 && at16(a.x), b = a.rank % 8 == 0;
    const bool y = a.ldy % 8 == 0 && at16(a.y) && at16(a.base);
    // (Ranks that are no multiple of 8, and rows off 16-byte boundaries, load by element.)
    if (x && b && y) launch_as<T, RT, true, true, true>(a, p, s);
    else if (x && y) launch_as<T, RT, true, false, true>(a, p, s);
    else if (b) launch_as<T, RT, false, true, false>(a, p, s);
    else launch_as<T, RT, false, false, false>(a, p, s);
}

template <class T> void launch_type(const AdapterArgs &a, const AdapterPlan &p, hipStream_t s) {
    if (a.rank <= 16) launch_rank<T, 1>(a, p, s);
    else if (a.rank <= 32) launch_rank<T, 2>(a, p, s);
    else if (a.rank <= 64) launch_rank<T, 4>(a, p, s);
    else launch_rank<T, 8>(a, p, s);
}

}  // namespace

size_t adapter_workspace_bytes(int rows, int adapters, int N, int K, int rank) {
    const AdapterPlan p = plan_adapter(rows, adapters, N, K, rank);
    const int pad = rank <= 32 ? 32 : rank <= 64 ? 64 : 128;
    return size_t(p.splits) * rows * pad * 4;
}

void launch_adapter(const AdapterArgs &a, hipStream_t s) {
    const AdapterPlan p = plan_adapter(a.rows, a.adapters, a.N, a.K, a.rank);
    if (a.type == F16) launch_type<f16_t>(a, p, s);
    else launch_type<bf16_t>(a, p, s);
}

}  // namespace qlin
