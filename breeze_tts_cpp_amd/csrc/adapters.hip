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
//
// Few rows: a chain of dependent loads (offsets, rows, A and x, B; 57 rows of 16
// adapters of rank 32, 12288 x 2048: 9.0 us, 1 row of rank 16, 4096 x 2048: 5.2). Many: the
// bytes of x, base and y (4096 rows of rank 64, 2048 x 6144: 29.3 us, 3.1 TB/s of 90 MB).
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

// Barrier for LDS alone: loads to LDS or registers stay in flight across it.
__device__ __forceinline__ void lds_barrier() {
    asm volatile("" ::: "memory");
    wait_lds_reads();  // (and writes)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// No memory access or other instruction is moved across.
__device__ __forceinline__ void pin() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The tile's row ml: its row of x and y, or -1.
__device__ __forceinline__ int source_row(const AdapterArgs &p, const RowTile &t, int ml) {
    int row = p.order[t.begin + min(ml, t.rows - 1)];
    asm("" : "+v"(row));  // (loaded without a branch, so that several loads go out together)
    return ml < t.rows && uint32_t(row) < uint32_t(p.rows) ? row : -1;
}
__device__ __forceinline__ int group_rank(const AdapterArgs &p, int g) {
    return p.ranks ? min(max(p.ranks[g], 0), p.rank) : p.rank;
}

// acc[i][t] += A rows r0 + [16 i, 16 i + 16) x the tile's tokens [16 t, 16 t + 16) over the
// wave's stages [k0, k0 + 64 count) of K; rows[i] is this lane's row of x in the tile's
// i-th eight. A fragment's lanes are 16 rows apart in memory, one cache line
// each: loaded straight to registers a CU takes in 32-45 B/ns. So a stage's rows of
// both operands go to the wave's own LDS first, 128 bytes (64 K) a row and eight
// lanes a line, chunk c of row r at c ^ ((r >> 1) & 7) (57 rows, 16 adapters of rank 16,
// 2048 x 6144: 12.7 -> 9.3 us). One stage a wave: with two to four in flight a decode
// call is no faster (6.4 us against 6.1) and fewer workgroups share a CU. Rows past
// the rank or the tile, and chunks past K, arrive as zeros. x that is not made of
// 16-byte pieces is copied there by element.
template <class T, int RT, int MT, int S, bool Vec>
__device__ __forceinline__ void shrink(const AdapterArgs &p, const RowTile &tile, int rank, int r0,
                                       const int (&rows)[2 * MT], int k0, int count, uint8_t *ring,
                                       f32x4 (&acc)[RT][MT]) {
    constexpr int BK = 128, STAGE = 16 * (RT + MT) * BK;
    static_assert(S == 1 || S == 2, "the waits below");
    constexpr uint32_t kOut = 0x80000000u;
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4, lane_row = lane >> 3;
    const uint32_t pitch = uint32_t(p.K) * 2u;
    const __amdgpu_buffer_rsrc_t rsrc_a = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint16_t *>(static_cast<const uint16_t *>(p.a) +
                               (size_t(tile.group) * p.rank + min(r0, p.rank - 1)) * p.K),
        0, max(rank - r0, 0) * int(pitch), 0x00020000);
    const __amdgpu_buffer_rsrc_t rsrc_x = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<void *>(p.x), 0, int((uint32_t(p.rows - 1) * uint32_t(p.ldx) + uint32_t(p.K)) * 2u),
        0x00020000);
    // A lane's chunk in instructions of even 8-row groups; 4 further in odd ones.
    const int chunk0 = (lane & 7) ^ (lane_row >> 1), chunk1 = chunk0 ^ 4;
    uint32_t xoff[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) {
        xoff[i] = rows[i] < 0 ? kOut : (uint32_t(rows[i]) * uint32_t(p.ldx) + uint32_t((i & 1 ? chunk1 : chunk0) * 8)) * 2u;
    }
    auto issue = [&](int st) {
        uint8_t *stage = ring + st % S * STAGE;
        const int k = k0 + st * 64;
        const bool in0 = k + chunk0 * 8 < p.K, in1 = k + chunk1 * 8 < p.K;
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
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
    pin();
#pragma unroll
    for (int s = 0; s < S; ++s)
        if (s < count) issue(s);
    for (int s = 0; s < count; ++s) {
        if (S == 2 && Vec && s + 1 < count) wait_vmcnt<2 * (RT + MT)>();
        else wait_vmcnt<0>();
        pin();
        const uint8_t *q = ring + s % S * STAGE + row16 * BK;
        uint4 av[RT][2], xv[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            xv[t][0] = *reinterpret_cast<const uint4 *>(q + (RT + t) * 16 * BK + c0);
            xv[t][1] = *reinterpret_cast<const uint4 *>(q + (RT + t) * 16 * BK + c1);
        }
#pragma unroll
        for (int i = 0; i < RT; ++i) {
            av[i][0] = *reinterpret_cast<const uint4 *>(q + i * 16 * BK + c0);
            av[i][1] = *reinterpret_cast<const uint4 *>(q + i * 16 * BK + c1);
        }
        pin();
        wait_lds_reads();
        pin();
        if (s + S < count) issue(s + S);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int t = 0; t < MT; ++t) mma16<T>(acc[i][t], av[i][h], xv[t][h]);
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
// Floats between two tokens of the waves' partial t: 16 tokens of a write on
// distinct banks (4096 rows of rank 64, 2048 x 6144: 38.5 -> 37.1 us).
constexpr int part_pitch(int rt) { return rank_pad(rt) + 4; }
constexpr int kAdapterWaves = 8, kAdapterThreads = 64 * kAdapterWaves;
constexpr int kPassChannels = 32 * kAdapterWaves;  // of the second product at a time
constexpr int kDeltaPitch = kPassChannels + 4;     // floats

// Two buffers of a pass's results.
constexpr int results_bytes(int mt) { return 2 * 16 * mt * kDeltaPitch * 4; }
// A single pass (Once) puts a wave's results, 32 channels of each token, where its
// B panel was, so that a CU takes three workgroups up to rank 64 (4096 rows of rank 64:
// 2048 x 6144 37.1 -> 35.2 us, 6144 x 2048 57 -> 46; of rank 128, with LDS for one, 39.4 ->
// 44.6: there a workgroup runs its passes in turn). Two lanes at most meet in a bank.
constexpr int kOncePitch = 36;  // floats
constexpr int once_bytes(int rp, int mt) {
    const int panel = 32 * rp * 2, results = 16 * mt * kOncePitch * 4;
    return (panel > results ? panel : results) + 128;
}

// The second product of the tile's 16 MT tokens for channels [n_begin, n_end), 256 at a time,
// 32 a wave: B's rows (one contiguous block of memory) through LDS like the
// operands above, the results through LDS to whole row pieces, so that base and y
// move in runs of 512 bytes. t is in hi / lo [16 MT][RP + 8]; `panel` holds 32 rows of B a
// wave, `results` two buffers of a pass's fp32 results (Once: not used).
template <class T, int RP, int MT, bool VecB, bool VecY, bool Once> struct Expand {
    // Rows of RP * 2 bytes, chunk c of row r at c ^ swizzle(r): fragment reads on
    // distinct banks. Chunks past the rank arrive as zeros; one that holds the
    // rank's end is cut when it is read.
    static constexpr int kChunks = RP / 8, kPanel = 32 * RP * 2;
    static constexpr int kStep = Once ? once_bytes(RP, MT) : kPanel;  // of the waves' LDS
    const AdapterArgs &p;
    const RowTile &tile;
    int rank, n_begin, n_end;
    uint8_t *panel;
    int to_row[MT], to_column;  // this thread's pieces of a pass's results: eight channels of a row

    __device__ __forceinline__ Expand(const AdapterArgs &p_, const RowTile &tile_, int rank_, int width,
                                      uint8_t *panels)
        : p(p_), tile(tile_), rank(rank_), n_begin(tile_.column * width),
          n_end(min(tile_.column * width + width, p_.N)),
          panel(panels + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kStep),
          to_column(threadIdx.x % 32 * 8) {
#pragma unroll
        for (int t = 0; t < MT; ++t) to_row[t] = source_row(p, tile, t * 16 + int(threadIdx.x) / 32);
    }
    static __device__ __forceinline__ int swizzle(int r) {
        return kChunks >= 8 ? (r >> 1 & 7) : (r * kChunks / 16) & (kChunks - 1);
    }
    __device__ __forceinline__ const uint16_t *rows_of_b(int n) const {
        return static_cast<const uint16_t *>(p.b) + (size_t(tile.group) * p.N + n) * p.rank;
    }
    // The wave's panel of the pass at n0.
    __device__ __forceinline__ void issue(int n0) const {
        if constexpr (VecB) {
            n0 = __builtin_amdgcn_readfirstlane(n0 + int(threadIdx.x >> 6) * 32);
            const int lane = threadIdx.x & 63;
            const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<uint16_t *>(rows_of_b(min(n0, p.N - 1))), 0,
                __builtin_amdgcn_readfirstlane(max(min(32, p.N - n0), 0) * p.rank * 2), 0x00020000);
#pragma unroll
            for (int i = 0; i < kPanel / 1024; ++i) {
                const int r = (i * 64 + lane) / kChunks, c = (i * 64 + lane) % kChunks ^ swizzle(r);
                const uint32_t at = c * 8 < rank ? uint32_t(r * p.rank + c * 8) * 2u : 0x80000000u;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)(panel + i * 1024), 16, at, 0, 0, 0);
            }
        }
    }
    // MFMA row i of fragment f is channel 8 (i / 4) + 4 f + i % 4 of the panel's 32, so
    // a lane's two fragments are eight consecutive channels of its token.
    __device__ __forceinline__ void read(int n0, uint4 (&o)[2][RP / 32]) const {
        const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            const int r = 8 * (row16 / 4) + 4 * f + row16 % 4;
#pragma unroll
            for (int s = 0; s < RP / 32; ++s) {
                const int c = s * 4 + quad, have = rank - c * 8;
                if constexpr (VecB) {
                    o[f][s] = *reinterpret_cast<const uint4 *>(panel + (r * kChunks + (c ^ swizzle(r))) * 16);
                } else {
                    const int n = n0 + int(threadIdx.x >> 6) * 32 + r;
                    o[f][s] = have > 0 && n < p.N ? load_piece(rows_of_b(n) + c * 8, have) : uint4{0, 0, 0, 0};
                }
            }
        }
    }
    // Panel fragments as read, with what lies past a rank in the middle of a piece cut off.
    __device__ __forceinline__ void cut(uint4 (&o)[2][RP / 32]) const {
        if (!VecB || rank % 8 == 0) return;
        const int quad = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
            for (int s = 0; s < RP / 32; ++s) o[f][s] = cut_piece(o[f][s], rank - (s * 4 + quad) * 8);
    }
    __device__ __forceinline__ void load_base(int n0, uint4 (&v)[MT]) const {
        const int n = n0 + to_column;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            v[t] = uint4{0, 0, 0, 0};
            if (p.base && to_row[t] >= 0 && n < n_end)
                v[t] = load_raw8<VecY>(static_cast<const uint16_t *>(p.base) + size_t(to_row[t]) * p.ldy + n, 0, 8);
        }
    }
    // All passes; the first panel is on its way, its base in `base`.
    __device__ __forceinline__ void run(const uint16_t *hi, const uint16_t *lo, const int *exponent,
                                        float *results, uint4 (&base)[MT]) const {
        constexpr int kPitch = RP + 8;
        const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
        const int wave = threadIdx.x >> 6;
        const float scale = p.scales ? p.scales[tile.group] : 1.f;
        int half = 0;
        for (int n0 = n_begin; n0 < n_end; n0 += kPassChannels, half ^= 1) {
            uint4 bv[2][RP / 32], next[MT];
            pin();
            wait_vmcnt<0>();  // the panel (and the base, asked for with it)
            pin();
            read(n0, bv);
            pin();
            wait_lds_reads();
            pin();
            cut(bv);
            if (!Once && n0 + kPassChannels < n_end) {
                issue(n0 + kPassChannels);
                load_base(n0 + kPassChannels, next);
            }
            // [token][channel of the pass or, once, of the wave]
            float *at = Once ? reinterpret_cast<float *>(panel)
                             : results + half * 16 * MT * kDeltaPitch + wave * 32;
            constexpr int kPitchOut = Once ? kOncePitch : kDeltaPitch;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                f32x4 out[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
                const int ml = t * 16 + row16, e = exponent[ml];
#pragma unroll
                for (int s = 0; s < RP / 32; ++s) {
                    const uint4 h = *reinterpret_cast<const uint4 *>(hi + ml * kPitch + s * 32 + quad * 8);
                    const uint4 l = *reinterpret_cast<const uint4 *>(lo + ml * kPitch + s * 32 + quad * 8);
#pragma unroll
                    for (int f = 0; f < 2; ++f) {
                        mma16<T>(out[f], bv[f][s], l);
                        mma16<T>(out[f], bv[f][s], h);
                    }
                }
#pragma unroll
                for (int f = 0; f < 2; ++f) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) out[f][r] = scale * __builtin_amdgcn_ldexpf(out[f][r], e);
                    *reinterpret_cast<f32x4 *>(at + ml * kPitchOut + quad * 8 + f * 4) = out[f];
                }
            }
            lds_barrier();  // (the other half was read before the last one)
            const int n = n0 + to_column;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                if (to_row[t] < 0 || n >= n_end) continue;
                const int ml = t * 16 + threadIdx.x / 32;
                const uint8_t *other = panel + (to_column / 32 - wave) * kStep;  // of the channels' wave
                const float *delta = Once ? reinterpret_cast<const float *>(other) + ml * kPitchOut + to_column % 32
                                          : at - wave * 32 + ml * kPitchOut + to_column;
                float v[8];
                widen8<T>(base[t], v);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += delta[i];
                store16x8<T, VecY>(static_cast<uint16_t *>(p.y) + size_t(to_row[t]) * p.ldy + n, 0, 8, v);
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) base[t] = next[t];
            if constexpr (Once) break;
        }
    }
};

// ---------------------------------------------------------------- one launch
// LDS: the waves' stages, then (their space again) the waves' partial sums of t,
// then the results; behind them the waves' B panels. Rank 128's stages leave the
// panels no room of their own: they lie behind the sums.
struct AdapterLds {
    int stage, panels_at, bytes;
};
constexpr AdapterLds adapter_lds(int rt) {
    AdapterLds l{};
    l.stage = 16 * (rt + 1) * 128;
    const int sums = kAdapterWaves * 16 * part_pitch(rt) * 4, results = results_bytes(1);
    const int reused = sums > results ? sums : results;
    const int stages = kAdapterWaves * l.stage;
    l.panels_at = rt == 8 || reused > stages ? reused : stages;
    l.bytes = l.panels_at + kAdapterWaves * 32 * rank_pad(rt) * 2;
    if (l.bytes < stages) l.bytes = stages;
    return l;
}

// One workgroup: 16 rows of one adapter, `width` channels. Its eight waves split
// K of the first product, sum t through LDS and take the second product's
// channels. Column tiles of the same rows repeat the first product.
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
    const int rows[2] = {source_row(p, tile, lane >> 3), source_row(p, tile, 8 + (lane >> 3))};
    const Expand<T, RP, 1, VecB, VecY, false> second(p, tile, rank, width, lds + kLds.panels_at);
    pin();
    if constexpr (RT < 8) second.issue(second.n_begin);

    f32x4 acc[RT][1];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i][0] = f32x4{0, 0, 0, 0};
    const int stages = (p.K + 63) / 64, each = (stages + W - 1) / W, first = min(wave * each, stages);
    shrink<T, RT, 1, 1, VecX>(p, tile, rank, 0, rows, first * 64, min(each, stages - first),
                           lds + wave * kLds.stage, acc);
    float *parts = reinterpret_cast<float *>(lds);
    __syncthreads();
    if constexpr (RT == 8) second.issue(second.n_begin);
#pragma unroll
    for (int i = 0; i < RP / 16; ++i)
        *reinterpret_cast<f32x4 *>(parts + (wave * 16 + row16) * part_pitch(RT) + i * 16 + quad * 4) =
            i < RT ? acc[i < RT ? i : 0][0] : f32x4{0, 0, 0, 0};
    __syncthreads();
    if (threadIdx.x < 256) {  // 16 lanes per token
        const int ml = threadIdx.x / 16, l = threadIdx.x % 16;
        float t[RP / 16];
#pragma unroll
        for (int i = 0; i < RP / 16; ++i) {
            t[i] = 0.f;
#pragma unroll
            for (int q = 0; q < W; ++q) t[i] += parts[(q * 16 + ml) * part_pitch(RT) + i * 16 + l];
            // (Past the rank A was read as zeros, but 0 * inf is NaN.)
            if (i * 16 + l >= rank) t[i] = 0.f;
        }
        split_token<T, RP>(t, hi + ml * kPitch, lo + ml * kPitch, exponent + ml);
    }
    uint4 base[1];
    second.load_base(second.n_begin, base);
    __syncthreads();
    second.run(hi, lo, exponent, reinterpret_cast<float *>(lds), base);
}

// ---------------------------------------------------------------- two launches
constexpr int kShrinkRows = 64, kExpandRows = 32, kShrinkWaves = 4, kMaxSplits = 4;
constexpr int shrink_lds_bytes(int rt) {
    const int rts = rt < 4 ? rt : 4, rings = kShrinkWaves * 2 * 16 * (rts + kShrinkRows / 16) * 128;
    const int sums = kShrinkWaves * kShrinkRows * part_pitch(rts) * 4;
    return rings > sums ? rings : sums;
}
// First product of a 64-row tile over one of `splits` ranges of K, which its four
// waves split, two stages in flight each; partial t [split][slot][RP] to the workspace. At most 64 ranks per
// workgroup.
template <class T, int RT, bool VecX>
__global__ __launch_bounds__(64 * kShrinkWaves) void adapter_shrink(AdapterArgs p, int splits) {
    constexpr int RP = rank_pad(RT), W = kShrinkWaves, MT = kShrinkRows / 16;
    constexpr int RTS = RT < 4 ? RT : 4, RPS = rank_pad(RTS), kParts = RP / RPS;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16 * MT, splits * kParts, blockIdx.x, tile)) return;
    const int lane = threadIdx.x & 63, row16 = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = tile.column / kParts, r0 = tile.column % kParts * RPS;
    const int rank = group_rank(p, tile.group);
    int rows[2 * MT];
#pragma unroll
    for (int i = 0; i < 2 * MT; ++i) rows[i] = source_row(p, tile, i * 8 + (lane >> 3));
    f32x4 acc[RTS][MT];
#pragma unroll
    for (int i = 0; i < RTS; ++i)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[i][t] = f32x4{0, 0, 0, 0};
    const int stages = (p.K + 63) / 64, each = (stages + W * splits - 1) / (W * splits);
    const int first = min((split * W + wave) * each, stages);
    shrink<T, RTS, MT, 2, VecX>(p, tile, rank, r0, rows, first * 64, min(each, stages - first),
                                lds + wave * 2 * 16 * (RTS + MT) * 128, acc);
    float *parts = reinterpret_cast<float *>(lds);
    float *out = static_cast<float *>(p.workspace) + (size_t(split) * p.rows + tile.begin) * RP + r0;
    __syncthreads();
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < RPS / 16; ++i)
            *reinterpret_cast<f32x4 *>(parts + ((wave * MT + t) * 16 + row16) * part_pitch(RTS) + i * 16 + quad * 4) =
                i < RTS ? acc[i < RTS ? i : 0][t] : f32x4{0, 0, 0, 0};
    __syncthreads();
    for (int i = threadIdx.x * 4; i < tile.rows * RPS; i += 64 * W * 4) {
        f32x4 s = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < W; ++q)
            s += *reinterpret_cast<const f32x4 *>(parts + (q * 16 * MT + i / RPS) * part_pitch(RTS) + i % RPS);
        *reinterpret_cast<f32x4 *>(out + size_t(i / RPS) * RP + i % RPS) = s;
    }
}

// Second product of a 32-row tile for `width` channels (LDS: panels, results).
template <class T, int RT, bool VecB, bool VecY>
__global__ __launch_bounds__(kAdapterThreads) void adapter_expand(AdapterArgs p, int splits, int columns,
                                                                  int width) {
    constexpr int RP = rank_pad(RT), MT = kExpandRows / 16, kPitch = RP + 8;
    constexpr bool kOnce = RT <= 4;
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];
    __shared__ __attribute__((aligned(16))) uint16_t hi[16 * MT * kPitch], lo[16 * MT * kPitch];
    __shared__ int exponent[16 * MT];
    RowTile tile;
    if (!find_tile(p.offsets, p.adapters, p.rows, 16 * MT, columns, blockIdx.x, tile)) return;
    const int rank = group_rank(p, tile.group);
    const Expand<T, RP, MT, VecB, VecY, kOnce> second(p, tile, rank, width, lds);
    second.issue(second.n_begin);
    uint4 base[MT];
    second.load_base(second.n_begin, base);
    static_assert(kAdapterThreads / 16 == 16 * MT, "16 lanes per token");
    const int ml = threadIdx.x / 16, l = threadIdx.x % 16;
    const float *t0 = static_cast<const float *>(p.workspace) +
                      (size_t(tile.begin) + min(ml, tile.rows - 1)) * RP + l;
    float t[RP / 16], u[kMaxSplits][RP / 16];
#pragma unroll
    for (int q = 0; q < kMaxSplits; ++q)
#pragma unroll
        for (int i = 0; i < RP / 16; ++i) u[q][i] = t0[size_t(min(q, splits - 1)) * p.rows * RP + i * 16];
#pragma unroll
    for (int i = 0; i < RP / 16; ++i) {
        t[i] = 0.f;
#pragma unroll
        for (int q = 0; q < kMaxSplits; ++q)
            if (q < splits && i * 16 + l < rank) t[i] += u[q][i];
    }
    split_token<T, RP>(t, hi + ml * kPitch, lo + ml * kPitch, exponent + ml);
    __syncthreads();
    second.run(hi, lo, exponent, reinterpret_cast<float *>(lds + kAdapterWaves * 32 * RP * 2), base);
}

// Splits of K of the two-launch form; 0: one launch, while the A matrices that its
// 16-row tiles read come to less than 32 MiB (rank 16: 48 MiB). One / two launches, us:
// 500 rows of 100 adapters of rank 64, 4096 x 2048, 31 MiB, 22.8 / 28.1; 1000 of 64 of rank
// 32, 4096 x 4096, 30 MiB, 15.6 / 17.9; 2048 of 8 of rank 32, 4096 x 4096, 34 MiB, 25.6 /
// 19.6; 4096 of 6 of rank 64, 6144 x 2048, 65 MiB, 72 / 43; rank 16: 8192 of 8, 2048 x 2048,
// 32 MiB, 24.6 / 30.0, 4096 of 6, 2048 x 6144, 49 MiB, 32.6 / 24.3. The 64-row tiles times
// the splits make one round of workgroups: in a second one 4096 rows of rank 64 take 44 us
// in place of 35 (two smaller workgroups per CU, 512 in a round, 38-40), of rank 128, 2048 x
// 2048, 40 in place of 37.
int plan_splits(int rows, int adapters, int K, int rank) {
    if (expert_row_tiles(rows, adapters, 16) * rank * K * 2 < (rank <= 16 ? 48L : 32L) << 20) return 0;
    const long groups = expert_row_tiles(rows, adapters, kShrinkRows) * (rank > 64 ? 2 : 1);
    return int(std::max(1L, std::min(std::min(256 / groups, long(kMaxSplits)), long(K) / 512)));
}

template <class T, int RT, bool VecX, bool VecB, bool VecY>
void launch_as(const AdapterArgs &a, hipStream_t s) {
    const int units = (a.N + kPassChannels - 1) / kPassChannels;
    // Column tiles of whole passes, as many as `wanted` workgroups need.
    auto width_of = [&](long tiles, long wanted) {
        const int most = int(std::max(1L, std::min(wanted / tiles, long(units))));
        return (units + most - 1) / most * kPassChannels;
    };
    if (const int splits = plan_splits(a.rows, a.adapters, a.K, a.rank)) {
        const long tiles = expert_row_tiles(a.rows, a.adapters, kShrinkRows);
        hipLaunchKernelGGL((adapter_shrink<T, RT, VecX>), dim3(unsigned(tiles * splits * (RT > 4 ? 2 : 1))),
                           dim3(64 * kShrinkWaves), shrink_lds_bytes(RT), s, a, splits);
        const long rows = expert_row_tiles(a.rows, a.adapters, kExpandRows);
        const int width = RT <= 4 ? kPassChannels : width_of(rows, 1024), columns = (a.N + width - 1) / width;
        constexpr int RP = rank_pad(RT), MT = kExpandRows / 16;
        constexpr int bytes = kAdapterWaves * (RT <= 4 ? once_bytes(RP, MT) : 32 * RP * 2) +
                              (RT <= 4 ? 0 : results_bytes(MT));
        static_assert(bytes + 4 * kExpandRows * (RP + 9) <= int(kLdsBytes), "LDS");
        hipLaunchKernelGGL((adapter_expand<T, RT, VecB, VecY>), dim3(unsigned(rows * columns)), dim3(kAdapterThreads),
                           bytes, s, a, splits, columns, width);
        return;
    }
    // Column tiles until the workgroups fill the CUs; of ranks up to 32, whose
    // operands leave the LDS room for three, three times once the row tiles are
    // many (4096 rows, rank 16, 4096 x 2048: 43 -> 25 us).
    const long tiles = expert_row_tiles(a.rows, a.adapters, 16);
    const int width = width_of(tiles, RT <= 2 && tiles > 128 ? 768 : 256);
    const int columns = (a.N + width - 1) / width;
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

size_t adapter_workspace_bytes(int rows, int adapters, int K, int rank) {
    const int pad = rank <= 32 ? 32 : rank <= 64 ? 64 : 128;
    return size_t(plan_splits(rows, adapters, K, rank)) * rows * pad * 4;
}

void launch_adapter(const AdapterArgs &a, hipStream_t s) {
    if (a.type == F16) launch_type<f16_t>(a, s);
    else launch_type<bf16_t>(a, s);
}

}  // namespace qlin
