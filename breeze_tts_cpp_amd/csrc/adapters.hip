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
// channels), the B operand 16 tokens, eight consecutive K values per lane; a
// lane's result is four consecutive A rows of one token.
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

// The first `have` of eight 16-bit values, zeros for the rest.
__device__ __forceinline__ uint4 cut_piece(const uint4 &v, int have) {
    auto keep = [&](uint32_t u, int i) { return have > i + 1 ? u : have > i ? u & 0xffffu : 0u; };
    return have >= 8 ? v : uint4{keep(v.x, 0), keep(v.y, 2), keep(v.z, 4), keep(v.w, 6)};
}
// Eight 16-bit values at p, zeros from `have` on, which are not read.
__device__ __forceinline__ uint4 load_piece(const uint16_t *p, int have) {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < have ? p[i] : 0;
    return uint4{e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16)};
}

// No memory access or other instruction is moved across.
__device__ __forceinline__ void pin() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
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

// acc[i] += A rows [16 i, 16 i + 16) x the tile's 16 tokens over the wave's stages
// [k0, k0 + 64 count) of K. A fragment's lanes are 16 rows apart in memory, one cache line
// each: loaded straight to registers a CU takes in 32-45 B/ns. So a stage's rows of
// both operands go to the wave's own LDS first, 128 bytes (64 K) a row and eight
// lanes a line, chunk c of row r at c ^ ((r >> 1) & 7) (57 rows, 16 adapters of rank 16,
// 2048 x 6144: 12.7 -> 9.3 us). One stage a wave: with two to four in flight a decode
// call is no faster (6.4 us against 6.1) and fewer workgroups share a CU. Rows past
// the rank or the tile, and chunks past K, arrive as zeros. x that is not made of
// 16-byte pieces is copied there by element.
template <class T, int RT, bool Vec>
__device__ __forceinline__ void shrink(const AdapterArgs &p, const RowTile &tile, int rank, int k0,
                                       int count, uint8_t *stage, f32x4 (&acc)[RT]) {
    constexpr int BK = 128;
    constexpr uint32_t kOut = 0x80000000u;
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4, lane_row = lane >> 3;
    const uint32_t pitch = uint32_t(p.K) * 2u;
    const __amdgpu_buffer_rsrc_t rsrc_a = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t *>(static_cast<const uint16_t *>(p.a) + size_t(tile.group) * p.rank * p.K), 0,
        rank * int(pitch), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsrc_x = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<void *>(p.x), 0, int((uint32_t(p.rows - 1) * uint32_t(p.ldx) + uint32_t(p.K)) * 2u),
        0x00020000);
    // A lane's chunk in instructions of even 8-row groups; 4 further in odd ones.
    const int chunk0 = (lane & 7) ^ (lane_row >> 1), chunk1 = chunk0 ^ 4;
    uint32_t xoff[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = source_row(p, tile, i * 8 + lane_row);
        xoff[i] = row < 0 ? kOut : (uint32_t(row) * uint32_t(p.ldx) + uint32_t((i & 1 ? chunk1 : chunk0) * 8)) * 2u;
    }
    auto issue = [&](int st) {
        const int k = k0 + st * 64;
        const bool in0 = k + chunk0 * 8 < p.K, in1 = k + chunk1 * 8 < p.K;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t at = (i & 1 ? in1 : in0) ? xoff[i] : kOut;
            if constexpr (Vec) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_x, (lds_ptr_t)(stage + (2 * RT + i) * 1024), 16, at,
                                                         uint32_t(k) * 2u, 0, 0);
            } else {
                uint4 v = uint4{0, 0, 0, 0};
                if (at != kOut) v = load_piece(static_cast<const uint16_t *>(p.x) + (at / 2 + uint32_t(k)), 8);
                *reinterpret_cast<uint4 *>(stage + (2 * RT + i) * 1024 + lane * 16) = v;
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * RT; ++i) {
            const uint32_t at = uint32_t(lane_row) * pitch + uint32_t((i & 1 ? chunk1 : chunk0) * 16);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_a, (lds_ptr_t)(stage + i * 1024), 16,
                                                     (i & 1 ? in1 : in0) ? at : kOut,
                                                     uint32_t(i) * 8u * pitch + uint32_t(k) * 2u, 0, 0);
        }
    };
    const int sw7 = (row16 >> 1) & 7, c0 = (quad ^ sw7) * 16, c1 = ((4 + quad) ^ sw7) * 16;
    const uint8_t *q = stage + row16 * BK;
    pin();
    if (count > 0) issue(0);
    for (int s = 0; s < count; ++s) {
        wait_vmcnt<0>();
        pin();
        uint4 av[RT][2], xv[2];
        xv[0] = *reinterpret_cast<const uint4 *>(q + RT * 16 * BK + c0);
        xv[1] = *reinterpret_cast<const uint4 *>(q + RT * 16 * BK + c1);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            av[i][0] = *reinterpret_cast<const uint4 *>(q + i * 16 * BK + c0);
            av[i][1] = *reinterpret_cast<const uint4 *>(q + i * 16 * BK + c1);
        }
        pin();
        wait_lds_reads();
        pin();
        if (s + 1 < count) issue(s + 1);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i) mma16<T>(acc[i], av[i][h], xv[h]);
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

constexpr int rank_pad(int rt) { return rt < 2 ? 32 : 16 * rt; }
constexpr int kAdapterWaves = 8, kAdapterThreads = 64 * kAdapterWaves;
constexpr int kPassChannels = 32 * kAdapterWaves;  // of the second product at a time
constexpr int kDeltaPitch = kPassChannels + 4;     // floats

// LDS: the waves' rings, then (their space again) the waves' partial sums of t,
// then two buffers of a pass's results; behind them the waves' B panels. Rank
// 128's rings leave the panels no room of their own: they lie behind the sums.
struct AdapterLds {
    int ring, panel, panels_at, bytes;
};
constexpr AdapterLds adapter_lds(int rt) {
    AdapterLds l{};
    l.ring = 16 * (rt + 1) * 128;
    l.panel = 32 * rank_pad(rt) * 2;
    const int sums = kAdapterWaves * 16 * rank_pad(rt) * 4, results = 2 * 16 * kDeltaPitch * 4;
    const int reused = sums > results ? sums : results;
    const int rings = kAdapterWaves * l.ring;
    l.panels_at = rt == 8 || reused > rings ? reused : rings;
    l.bytes = l.panels_at + kAdapterWaves * l.panel;
    if (l.bytes < rings) l.bytes = rings;
    return l;
}

// One workgroup: 16 rows of one adapter, `width` channels. Its eight waves split
// K of the first product and sum t through LDS, which is split into hi and lo
// there. Then they take 256 channels at a time of the second, 32 each: B's rows
// (one contiguous block of memory) through LDS like the operands above, the
// results through LDS to whole row pieces, so that base and y move in runs of
// 512 bytes. Column tiles of the same rows repeat the first product.
template <class T, int RT, bool VecX, bool VecB, bool VecY>
__global__ __launch_bounds__(kAdapterThreads) void adapter_rows(AdapterArgs p, int columns, int width) {
    constexpr int RP = rank_pad(RT), W = kAdapterWaves, kPitch = RP + 8;
    constexpr AdapterLds kLds = adapter_lds(RT);
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ __attribute__((aligned(16))) uint16_t hi[16 * kPitch], lo[16 * kPitch];
    __shared__ int exponent[16];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16, columns, blockIdx.x, tile)) return;
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rank = group_rank(p, tile.group);
    const float scale = p.scales ? p.scales[tile.group] : 1.f;
    const int n_begin = tile.column * width, n_end = min(n_begin + width, p.N);

    // B's panel of 32 channels, rows of RP * 2 bytes, chunk c of row r at c ^
    // ((r * chunks / 8) % chunks): fragment reads on distinct banks. Chunks past the
    // rank arrive as zeros; one that holds the rank's end is cut when it is read.
    constexpr int kChunks = RP / 8;
    uint8_t *panel = lds + kLds.panels_at + wave * kLds.panel;
    auto swizzle = [&](int r) { return kChunks >= 8 ? (r >> 1 & 7) : (r * kChunks / 16) & (kChunks - 1); };
    const uint16_t *b_group = static_cast<const uint16_t *>(p.b) + size_t(tile.group) * p.N * p.rank;
    auto issue_panel = [&](int n0) {
        if constexpr (VecB) {
            const int rows = max(min(32, p.N - n0), 0);
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint16_t *>(b_group + size_t(min(n0, p.N - 1)) * p.rank), 0, rows * p.rank * 2,
                0x00020000);
#pragma unroll
            for (int i = 0; i < kLds.panel / 1024; ++i) {
                const int r = (i * 64 + lane) / kChunks, c = (i * 64 + lane) % kChunks ^ swizzle(r);
                const uint32_t at = c * 8 < rank ? uint32_t(r * p.rank + c * 8) * 2u : 0x80000000u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(panel + i * 1024), 16, at, 0, 0, 0);
            }
        }
    };
    // MFMA row r of fragment f is channel 8 (r / 4) + 4 f + r % 4 of the panel's 32, so
    // a lane's two fragments are eight consecutive channels of its token.
    auto read_panel = [&](int n0, uint4 (&o)[2][RP / 32]) {
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const int r = 8 * (row16 / 4) + 4 * f + row16 % 4;
#pragma unroll
            for (int s = 0; s < RP / 32; ++s) {
                const int c = s * 4 + quad, have = rank - c * 8;
                if constexpr (VecB) {
                    o[f][s] = *reinterpret_cast<const uint4 *>(panel + (r * kChunks + (c ^ swizzle(r))) * 16);
                    o[f][s] = cut_piece(o[f][s], have);
                } else {
                    o[f][s] = uint4{0, 0, 0, 0};
                    if (have > 0 && n0 + r < p.N)
                        o[f][s] = load_piece(b_group + size_t(n0 + r) * p.rank + c * 8, have);
                }
            }
        }
    };
    if constexpr (RT < 8) issue_panel(n_begin + wave * 32);

    f32x4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = f32x4{0, 0, 0, 0};
    const int stages = (p.K + 63) / 64, each = (stages + W - 1) / W, first = min(wave * each, stages);
    shrink<T, RT, VecX>(p, tile, rank, first * 64, min(each, stages - first),
                                        lds + wave * kLds.ring, acc);
    float *parts = reinterpret_cast<float *>(lds);
    __syncthreads();
    if constexpr (RT == 8) issue_panel(n_begin + wave * 32);
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
    // This thread's piece of a pass's results: eight channels of one row.
    const int to_row = source_row(p, tile, threadIdx.x / 32), to_column = threadIdx.x % 32 * 8;
    auto load_base = [&](int n0) {
        const int n = n0 + to_column;
        uint4 v = uint4{0, 0, 0, 0};
        if (p.base && to_row >= 0 && n < n_end)
            v = load_raw8<VecY>(static_cast<const uint16_t *>(p.base) + size_t(to_row) * p.ldy + n, 0, 8);
        return v;
    };
    uint4 base = load_base(n_begin);
    __syncthreads();
    uint4 h[RP / 32], l[RP / 32];
#pragma unroll
    for (int s = 0; s < RP / 32; ++s) {
        h[s] = *reinterpret_cast<const uint4 *>(hi + row16 * kPitch + s * 32 + quad * 8);
        l[s] = *reinterpret_cast<const uint4 *>(lo + row16 * kPitch + s * 32 + quad * 8);
    }
    const int e = exponent[row16];
    float *results = reinterpret_cast<float *>(lds);
    int half = 0;
    for (int n0 = n_begin; n0 < n_end; n0 += kPassChannels, half ^= 1) {
        uint4 bv[2][RP / 32];
        pin();
        wait_vmcnt<0>();  // the panel (and the base, asked for with it)
        pin();
        read_panel(n0 + wave * 32, bv);
        pin();
        wait_lds_reads();
        pin();
        uint4 next_base = uint4{0, 0, 0, 0};
        if (n0 + kPassChannels < n_end) {
            issue_panel(n0 + kPassChannels + wave * 32);
            next_base = load_base(n0 + kPassChannels);
        }
        f32x4 out[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
        for (int s = 0; s < RP / 32; ++s)
#pragma unroll
            for (int f = 0; f < 2; ++f) {
                mma16<T>(out[f], bv[f][s], l[s]);
                mma16<T>(out[f], bv[f][s], h[s]);
            }
        float *at = results + half * 16 * kDeltaPitch;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
#pragma unroll
            for (int r = 0; r < 4; ++r) out[f][r] = scale * __builtin_amdgcn_ldexpf(out[f][r], e);
            *reinterpret_cast<f32x4 *>(at + row16 * kDeltaPitch + wave * 32 + quad * 8 + f * 4) = out[f];
        }
        __syncthreads();  // (the other half was read before the last one)
        const int n = n0 + to_column;
        if (to_row >= 0 && n < n_end) {
            const float *delta = at + threadIdx.x / 32 * kDeltaPitch + to_column;
            float v[8];
            widen8<T>(base, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += delta[i];
            store16x8<T, VecY>(static_cast<uint16_t *>(p.y) + size_t(to_row) * p.ldy + n, 0, 8, v);
        }
        base = next_base;
    }
}

template <class T, int RT, bool VecX, bool VecB, bool VecY>
void launch_as(const AdapterArgs &a, hipStream_t s) {
    // Column tiles until the workgroups fill the CUs; of ranks up to 32, whose
    // operands leave the LDS room for three, three times once the row tiles are
    // many (4096 rows, rank 16, 4096 x 2048: 43 -> 25 us).
    const long tiles = expert_row_tiles(a.rows, a.adapters, 16), wanted = RT <= 2 && tiles > 128 ? 768 : 256;
    const int units = (a.N + kPassChannels - 1) / kPassChannels;
    const int most = int(std::max(1L, std::min(wanted / tiles, long(units))));
    const int width = (units + most - 1) / most * kPassChannels, columns = (a.N + width - 1) / width;
    constexpr AdapterLds kLds = adapter_lds(RT);
    static_assert(kLds.bytes + 2 * 16 * (rank_pad(RT) + 8) * 2 + 64 <= int(kLdsBytes), "LDS");
    hipLaunchKernelGGL((adapter_rows<T, RT, VecX, VecB, VecY>), dim3(unsigned(tiles * columns)),
                       dim3(kAdapterThreads), kLds.bytes, s, a, columns, width);
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
