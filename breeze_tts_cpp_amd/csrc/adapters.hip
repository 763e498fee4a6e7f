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

// acc[i] += A rows [16 i, 16 i + 16) x the tile's 16 tokens over K [k0, k1). A block is 64 K: a
// lane takes 16 of them for two MFMAs (both operands in the same order), so its
// two loads and its row's four lanes cover a whole 128-byte line. `Deep` blocks
// are asked for ahead of the ones multiplied.
template <class T, int RT, int Deep, bool Vec>
__device__ __forceinline__ void shrink(const AdapterArgs &p, const RowTile &tile, int rank, int row,
                                       int k0, int k1, f32x4 (&acc)[RT]) {
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
    const uint16_t *xrow = static_cast<const uint16_t *>(p.x) + size_t(max(row, 0)) * p.ldx;
    const uint16_t *arow[RT];
    bool ain[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int r = i * 16 + row16;
        ain[i] = r < rank;
        arow[i] = static_cast<const uint16_t *>(p.a) +
                  (size_t(tile.group) * p.rank + min(r, p.rank - 1)) * p.K;
    }
    struct Block {
        uint4 x[2], a[RT][2];
    };
    // Pieces past the range come from the row's start and count as zeros.
    auto load = [&](int k, Block &o) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = k + quad * 16 + h * 8;
            const bool in = at < k1;
            const uint4 none = uint4{0, 0, 0, 0};
            const uint4 xv = load_piece<Vec>(xrow + (in ? at : 0), 8);
            o.x[h] = in && row >= 0 ? xv : none;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                const uint4 av = load_piece<true>(arow[i] + (in ? at : 0), 8);
                o.a[i][h] = in && ain[i] ? av : none;
            }
        }
    };
    auto multiply = [&](const Block &o) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i) mma16<T>(acc[i], o.a[i][h], o.x[h]);
    };
    Block now[Deep], next[Deep];
#pragma unroll
    for (int d = 0; d < Deep; ++d) load(k0 + d * 64, now[d]);
    for (int k = k0; k < k1; k += Deep * 64) {
        const bool more = k + Deep * 64 < k1;
        if (more) {
#pragma unroll
            for (int d = 0; d < Deep; ++d) load(k + (Deep + d) * 64, next[d]);
        }
#pragma unroll
        for (int d = 0; d < Deep; ++d) multiply(now[d]);
#pragma unroll
        for (int d = 0; d < Deep; ++d) now[d] = next[d];
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

// What the second product reads for channels [n0, n0 + 32): B's rows and the
// base. MFMA row p of fragment f is channel 8 (p / 4) + 4 f + p % 4 of the 32,
// so a lane's two fragments are eight consecutive channels of its token.
template <int RP> struct Panel {
    uint4 b[2][RP / 32], base;
};
template <class T, int RP, bool VecB, bool VecY>
__device__ __forceinline__ void load_panel(const AdapterArgs &p, const RowTile &tile, int rank, int row,
                                           int n0, Panel<RP> &o) {
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
#pragma unroll
    for (int f = 0; f < 2; ++f) {
        const int n = n0 + 8 * (row16 / 4) + 4 * f + row16 % 4;
        const uint16_t *at = static_cast<const uint16_t *>(p.b) +
                             (size_t(tile.group) * p.N + min(n, p.N - 1)) * p.rank;
#pragma unroll
        for (int s = 0; s < RP / 32; ++s) {
            const int r = s * 32 + quad * 8;
            const int have = n < p.N ? min(rank - r, 8) : 0;
            o.b[f][s] = have > 0 ? load_piece<VecB>(at + r, have) : uint4{0, 0, 0, 0};
        }
    }
    const int n = n0 + quad * 8;
    o.base = uint4{0, 0, 0, 0};
    if (p.base && row >= 0 && n < p.N)
        o.base = load_raw8<VecY>(static_cast<const uint16_t *>(p.base) + size_t(row) * p.ldy + n, 0, 8);
}

constexpr int rank_pad(int rt) { return rt < 2 ? 32 : 16 * rt; }
constexpr int kAdapterWaves = 8, kAdapterThreads = 64 * kAdapterWaves;

// One workgroup: 16 rows of one adapter, `width` channels. Its eight waves split
// K of the first product, sum t through LDS, split it into hi and lo there, and
// take 32 channels at a time of the second, the next 32's operands (the first
// ones from the start) asked for ahead. Column tiles of the same rows repeat the
// first product.
template <class T, int RT, bool VecX, bool VecB, bool VecY>
__global__ __launch_bounds__(kAdapterThreads) void adapter_rows(AdapterArgs p, int columns, int width) {
    constexpr int RP = rank_pad(RT), W = kAdapterWaves, kPitch = RP + 8;
    constexpr int Deep = RT >= 4 ? 1 : RT == 2 ? 2 : 4;
    __shared__ __attribute__((aligned(16))) float parts[W * 16 * RP];
    __shared__ __attribute__((aligned(16))) uint16_t hi[16 * kPitch], lo[16 * kPitch];
    __shared__ int exponent[16];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16, columns, blockIdx.x, tile)) return;
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rank = group_rank(p, tile.group);
    const float scale = p.scales ? p.scales[tile.group] : 1.f;
    const int row = source_row(p, tile, row16);
    const int n_first = tile.column * width + wave * 32;
    const int n_end = min((tile.column + 1) * width, p.N);
    Panel<RP> now, next;
    load_panel<T, RP, VecB, VecY>(p, tile, rank, row, min(n_first, p.N - 1), now);

    f32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    const int span = ((p.K + 63) / 64 + W - 1) / W * 64;
    const int k0 = min(wave * span, p.K);
    shrink<T, RT, Deep, VecX>(p, tile, rank, row, k0, min(k0 + span, p.K), acc);
#pragma unroll
    for (int i = 0; i < RP / 16; ++i)
        *reinterpret_cast<f32x4 *>(parts + (wave * 16 + row16) * RP + i * 16 + quad * 4) =
            i < RT ? acc[i < RT ? i : 0] : f32x4{0, 0, 0, 0};
    __syncthreads();
    if (threadIdx.x < 256) {  // 16 lanes per token
        const int ml = threadIdx.x / 16, l = threadIdx.x % 16;
        float t[RP / 16];
#pragma unroll
        for (int i = 0; i < RP / 16; ++i) {
            t[i] = 0.f;
#pragma unroll
            for (int q = 0; q < W; ++q) t[i] += parts[(q * 16 + ml) * RP + i * 16 + l];
            // (Past the rank A was read as zeros, but 0 * inf is NaN.)
            if (i * 16 + l >= rank) t[i] = 0.f;
        }
        split_token<T, RP>(t, hi + ml * kPitch, lo + ml * kPitch, exponent + ml);
    }
    __syncthreads();
    uint4 h[RP / 32], l[RP / 32];
#pragma unroll
    for (int s = 0; s < RP / 32; ++s) {
        h[s] = *reinterpret_cast<const uint4 *>(hi + row16 * kPitch + s * 32 + quad * 8);
        l[s] = *reinterpret_cast<const uint4 *>(lo + row16 * kPitch + s * 32 + quad * 8);
    }
    const int e = exponent[row16];
    for (int n0 = n_first; n0 < n_end; n0 += W * 32) {
        if (n0 + W * 32 < n_end) load_panel<T, RP, VecB, VecY>(p, tile, rank, row, n0 + W * 32, next);
        f32x4 out[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int s = 0; s < RP / 32; ++s)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                mma16<T>(out[f], now.b[f][s], l[s]);
                mma16<T>(out[f], now.b[f][s], h[s]);
            }
        float v[8];
        widen8<T>(now.base, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += scale * __builtin_amdgcn_ldexpf(out[i / 4][i % 4], e);
        const int n = n0 + quad * 8;
        if (row >= 0 && n < p.N)
            store16x8<T, VecY>(static_cast<uint16_t *>(p.y) + size_t(row) * p.ldy + n, 0, 8, v);
        now = next;
    }
}

template <class T, int RT, bool VecX, bool VecB, bool VecY>
void launch_as(const AdapterArgs &a, hipStream_t s) {
    // Column tiles until the row tiles fill the CUs, of at least 256 channels.
    const long tiles = expert_row_tiles(a.rows, a.adapters, 16);
    const int units = (a.N + 255) / 256;
    const int wanted = int(std::max(1L, std::min(256 / tiles, long(units))));
    const int width = (units + wanted - 1) / wanted * 256, columns = (a.N + width - 1) / width;
    hipLaunchKernelGGL((adapter_rows<T, RT, VecX, VecB, VecY>), dim3(unsigned(tiles * columns)),
                       dim3(kAdapterThreads), 0, s, a, columns, width);
}

template <class T, int RT>
void launch_rank(const AdapterArgs &a, hipStream_t s) {
    auto at16 = [](const void *q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
    const bool x = a.ldx % 8 == 0 && at16(a.x), b = a.rank % 8 == 0;
    const bool y = a.ldy % 8 == 0 && at16(a.y) && at16(a.base);
    // (Ranks that are no multiple of 8, and rows off 16-byte boundaries, load by element.)
    if (x && b && y) launch_as<T, RT, true, true, true>(a, s);
    else if (x && y) launch_as<T, RT, true, false, true>(a, s);
    else if (b) launch_as<T, RT, false, true, false>(a, s);
    else launch_as<T, RT, false, false, false>(a, s);
}

template <class T> void launch_type(const AdapterArgs &a, hipStream_t s) {
    if (a.rank <= 16) launch_rank<T, 1>(a, s);
    else if (a.rank <= 32) launch_rank<T, 2>(a, s);
    else if (a.rank <= 64) launch_rank<T, 4>(a, s);
    else launch_rank<T, 8>(a, s);
}

}  // namespace

void launch_adapter(const AdapterArgs &a, hipStream_t s) {
    if (a.type == F16) launch_type<f16_t>(a, s);
    else launch_type<bf16_t>(a, s);
}

}  // namespace qlin
