// Quantized products of rows grouped by expert (qlin_expert_gemm) for gfx950:
// y[s, :] = D(dequant(x[r(s)] . w[e(s)]^T)) for the slots s of each expert e's
// range of `offsets`; r(s) = order ? order[s] / divisor : s, the result row s or
// (scatter) order[s]. INT8 (exact int32) or FP8 codes, per-channel scales
// ((acc * sx) * sw) or K groups of 128 (fma(p_g, sx_g * sw_g, r), ascending g).
//
// The groups' sizes are known on the device only: the grid is the host's
// upper bound on macro tiles and each workgroup finds its tile (find_tile).
//
// Structure: KS slices of K times WN x WM waves. Each slice has an LDS ring of S
// stages (BN weight rows and BM token rows of 128 K bytes) filled by
// buffer_load ... lds; the token rows are gathered there, a lane's row offset
// held in a register for the whole walk. Rows past the group and chunks past K
// arrive as zeros (out-of-range offsets). The partial tiles of the slices are
// summed through LDS in ascending slice order.
//
// Bound by the live experts' weights while an expert has few rows (192 slots of 64
// experts, 2048 x 1024 FP8: 21.6 us, 5.2 TB/s with what the Infinity Cache gives; 8 of 64, 2048 x
// 2048 INT8: 7.7 us, 4.4 TB/s). With many no part alone is the bound: 16384 slots of 32
// experts, 4096 x 2048 INT8, take 158 us where the routing's tiles fill five rounds of
// workgroups, 178-186 where they begin a sixth (1.5-1.74 POPS; 2.0 at 4096 rows each). Of 167
// us on average 142 stay without the MFMAs, 136 without the loads past the first stages, 155
// without fragment reads or without stores, 85 without MFMAs and loads, 58 with prologue,
// barriers and epilogue alone. Between them a workgroup's fixed part is the most (7680 slots of
// 64, 2048 x 1024 FP8 with K groups, 57 us, 570 TFLOPS: 53 without MFMAs, fragment reads or
// stores, 43 without the loads past the first stages, 27 without the walk over K).
#include "qlin_device.hpp"
#include "qlin_internal.hpp"
#include "row_groups.hpp"

#include <algorithm>
#include <type_traits>

namespace qlin {
#ifdef QLIN_EXPERT_PART
namespace {

// A stage: its rows and, with K groups, 1 KB of channel scales, the tokens' scales and
// 256 bytes that surplus scale loads write.
constexpr int expert_stage_bytes(bool grouped, int bn, int bm) {
    return (bn + bm) * 128 + (grouped ? 1024 + (bm + 63) / 64 * 256 + 256 : 0);
}
// LDS of the slices' rings; afterwards of the partial tiles (one slice: of the
// 16-bit results).
constexpr int expert_body_bytes(bool grouped, int slices, int stages, int bn, int bm) {
    const int ring = slices * stages * expert_stage_bytes(grouped, bn, bm);
    const int sums = slices == 1 ? bm * (bn + 8) * 2 : slices * bm * (bn + 4) * 4;
    return ring > sums ? ring : sums;
}

// No memory access or other instruction is moved across.
__device__ __forceinline__ void pin() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// S = 2 (per-channel scales): a stage is refilled in halves (half_steps).
template <int Fmt, bool Grouped, int KS, int WN, int WM, int NF, int MT, int S, int EU>
__global__ __launch_bounds__(64 * KS * WN * WM, EU) void expert_gemm(ExpertArgs p, int tiles_n,
                                                                     int steps) {
    using Mma = TileMma<Fmt>;
    using Acc = typename Mma::Acc;
    constexpr int NWS = WN * WM, W = KS * NWS;
    constexpr int BN = 16 * NF * WN, BM = 16 * MT * WM, BK = 128;
    constexpr int STAGE = expert_stage_bytes(Grouped, BN, BM);
    // DMA instructions per wave and stage: weight rows, token rows and (K groups)
    // scales, of which instruction 0 is the channels' and q the tokens [64 (q - 1), ..).
    constexpr int SI = Grouped ? (1 + (BM + 63) / 64 + NWS - 1) / NWS : 0;
    constexpr int WI = BN / 8 / NWS, XI = BM / 8 / NWS, INSTS = WI + XI + SI;
    static_assert(BN / 8 % NWS == 0 && BM / 8 % NWS == 0, "whole DMA instructions per wave");
    static_assert(S > 1 && (NWS == 1 || NWS % 2 == 0), "the ring refills behind its readers");
    extern __shared__ __attribute__((aligned(1024))) uint8_t lds[];

    RowTile tile;
    if (!find_tile(p.offsets, p.experts, p.slots, BM, tiles_n, blockIdx.x, tile)) return;
    const int K = p.K, N = p.N, n_base = tile.column * BN, m_base = tile.begin;
    const uint8_t *w = p.w + size_t(tile.group) * N * K;
    const int k_groups = (K + 127) / 128;
    const float *sw = p.sw + size_t(tile.group) * N * (Grouped ? k_groups : 1);

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int row16 = lane & 15, quad = lane >> 4;
    const int ks = wave / NWS, ws = wave % NWS, wn = ws % WN, wm = ws / WN;
    // The tile's row ml in x, or -1 (past the group, or an order entry outside x), in
    // two parts: the load, which other loads need not wait for (without an order
    // it reads an offset), and the row.
    const int *entries = p.order ? p.order + m_base : p.offsets;
    auto entry = [&](int ml) { return entries[p.order ? min(ml, tile.rows - 1) : 0]; };
    auto source = [&](int at, int ml) {
        const int row = p.order ? int(uint32_t(at) / uint32_t(p.divisor)) : m_base + ml;
        return ml < tile.rows && (!p.order || at >= 0) && row < p.x_rows ? row : -1;
    };

    const int k_begin = ks * steps * BK;
    const int count = NWS > 1 ? steps : max(0, min(steps, (K - k_begin + BK - 1) / BK));
    const int rows_w = min(BN, N - n_base);
    const __amdgpu_buffer_rsrc_t rsrc_w = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(w + size_t(n_base) * K), 0, rows_w * K, 0x00020000);
    // Gathered rows: offsets from x (the host holds x_rows * K below 2^31); rows
    // in slot order: from the tile's first row.
    const __amdgpu_buffer_rsrc_t rsrc_x = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<uint8_t *>(p.order ? p.x : p.x + size_t(m_base) * K), 0,
        p.order ? p.x_rows * K : tile.rows * K, 0x00020000);
    // One DMA instruction fills 8 stage rows of 128 bytes in lane order; row r
    // keeps 16-byte chunk c at c ^ ((r >> 1) & 7) (fragment reads on distinct
    // banks), so a lane's source chunk goes by the parity of the instruction's
    // 8-row group (with a shared ring the same for all the wave's).
    const int lane_row = lane >> 3;
    const int chunk0 = (lane & 7) ^ (lane_row >> 1) ^ (NWS > 1 ? 4 * (ws & 1) : 0);
    const int chunk1 = chunk0 ^ 4;
    const uint32_t woff0 = uint32_t(lane_row) * uint32_t(K) + uint32_t(chunk0 * 16);
    const uint32_t woff1 = uint32_t(lane_row) * uint32_t(K) + uint32_t(chunk1 * 16);
    constexpr uint32_t kOut = 0x80000000u;  // an offset past every buffer: reads as zero
    auto x_ml = [&](int i) { return (NWS > 1 ? i * NWS + ws : i) * 8 + lane_row; };
    auto s_ml = [&](int i) { return (i * NWS + ws - 1) * 64 + lane; };
    int x_entry[XI], s_entry[SI + 1], to_entry = entry(tid);
#pragma unroll
    for (int i = 0; i < XI; ++i) x_entry[i] = entry(x_ml(i));
#pragma unroll
    for (int i = 0; i < SI; ++i) s_entry[i] = entry(max(s_ml(i), 0));
    uint8_t *ring = lds + ks * S * STAGE;
    uint8_t *dma_base = ring;
    uint32_t dk = 0;
    bool in0 = true, in1 = true;
    auto aim = [&](int st, int slot) {
        dma_base = ring + slot * STAGE;
        dk = uint32_t(k_begin + st * BK);
        in0 = st < count && int(dk) + chunk0 * 16 < K, in1 = st < count && int(dk) + chunk1 * 16 < K;
    };
    auto dma_w = [&](auto j_) {
        constexpr int j = decltype(j_)::value;
        const int g = NWS > 1 ? j * NWS + ws : j;  // 8-row group of the operand
        const bool odd = NWS == 1 && (j & 1);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rsrc_w, (lds_ptr_t)(dma_base + g * 1024), 16, (odd ? in1 : in0) ? (odd ? woff1 : woff0) : kOut,
            uint32_t(g) * 8u * uint32_t(K) + dk, 0, 0);
    };
    uint32_t xoff[XI];
    auto dma_x = [&](auto j_) {
        constexpr int j = decltype(j_)::value;
        const int g = NWS > 1 ? j * NWS + ws : j;
        const uint32_t at = (NWS == 1 && (j & 1) ? in1 : in0) ? xoff[j] : kOut;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_x, (lds_ptr_t)(dma_base + (BN / 8 + g) * 1024), 16, at,
                                                 dk, 0, 0);
    };
    // The first S stages: their weights are asked for before the rows' addresses
    // are known (those wait for the offsets, then the order). Stages that the slice
    // does not have are asked for as zeros, so that every wave's count of loads in
    // flight is known and no wait is longer than it has to be.
    pin();
#pragma unroll
    for (int s = 0; s < S; ++s) {
        aim(s, s);
        static_for<0, WI>(dma_w);
    }
    pin();
#pragma unroll
    for (int i = 0; i < XI; ++i) {
        const int chunk = NWS > 1 || !(i & 1) ? chunk0 : chunk1, row = source(x_entry[i], x_ml(i));
        xoff[i] = row < 0 ? kOut
                          : uint32_t(p.order ? row : row - m_base) * uint32_t(K) + uint32_t(chunk * 16);
    }

    // K groups: a stage's scales arrive with it, [BN] then [BM] floats behind its
    // rows, the tokens' gathered like the rows. Instructions that a wave has
    // beside these write zeros behind them (all waves count the same loads).
    const __amdgpu_buffer_rsrc_t rsrc_sw = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float *>(sw + n_base), 0, Grouped ? (k_groups * N - n_base) * 4 : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t rsrc_sx = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<float *>(p.sx), 0, Grouped ? k_groups * p.x_rows * 4 : 0, 0x00020000);
    uint32_t soff[SI + 1];
#pragma unroll
    for (int i = 0; i < SI; ++i) {
        const int q = i * NWS + ws, ml = s_ml(i);
        const int row = q > 0 && ml < BM ? source(s_entry[i], ml) : -1;
        soff[i] = q == 0 ? (lane * 4 < BN && n_base + lane * 4 < N ? uint32_t(lane * 16) : kOut)
                  : row < 0 ? kOut : uint32_t(row) * 4u;
    }
    auto dma_s = [&](auto i_) {
        constexpr int i = decltype(i_)::value;
        const uint32_t g = dk / BK, at = int(g) < k_groups ? soff[i] : kOut;
        const int q = i * NWS + ws;
        uint8_t *dst = dma_base + (BN + BM) * BK;
        if (q == 0) {
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_sw, (lds_ptr_t)dst, 16, at, g * uint32_t(N) * 4u, 0, 0);
        } else {
            dst += 1024 + min(q - 1, (BM + 63) / 64) * 256;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc_sx, (lds_ptr_t)dst, 4, at,
                                                     g * uint32_t(p.x_rows) * 4u, 0, 0);
        }
    };
    auto dma = [&](auto i_) {
        constexpr int i = decltype(i_)::value;
        if constexpr (i < WI) dma_w(std::integral_constant<int, i < WI ? i : 0>{});
        else if constexpr (i < WI + XI) dma_x(std::integral_constant<int, i < WI ? 0 : i - WI>{});
        else dma_s(std::integral_constant<int, i < WI + XI ? 0 : i - WI - XI>{});
    };

    // For the epilogue: a row's scale and where it goes, a channel's scale, one each
    // per thread until the walk is done (a wait for them here would wait for the
    // weights), then in LDS past the ring.
    static_assert(BM <= 64 * W && BN <= 64 * W, "one row and one channel per thread");
    constexpr int kBody = expert_body_bytes(Grouped, KS, S, BN, BM);
    float *row_scale = reinterpret_cast<float *>(lds + kBody), *col_scale = row_scale + BM;
    int *row_to = reinterpret_cast<int *>(col_scale + BN);
    const float row_scale_v = Grouped ? 1.f : p.sx[max(source(to_entry, tid), 0)];
    const float col_scale_v = Grouped ? 1.f : sw[min(n_base + tid, N - 1)];

    using Sum = std::conditional_t<Grouped, f32x4, Acc>;
    Sum acc[NF][MT];
#pragma unroll
    for (int f = 0; f < NF; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = Sum{0, 0, 0, 0};

    const int sw7 = (row16 >> 1) & 7;
    const int c0 = (quad ^ sw7) * 16, c1 = ((4 + quad) ^ sw7) * 16;
    auto frag = [&](int slot, int row) {
        const uint8_t *q = ring + slot * STAGE + (row + row16) * BK;
        const i32x4 lo = *reinterpret_cast<const i32x4 *>(q + c0);
        const i32x4 hi = *reinterpret_cast<const i32x4 *>(q + c1);
        return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto read_x = [&](int slot, auto &b) {
#pragma unroll
        for (int t = 0; t < int(sizeof(b) / sizeof(b[0])); ++t) b[t] = frag(slot, BN + (t * WM + wm) * 16);
    };
    auto read_w = [&](int slot, int f) { return frag(slot, (f * WN + wn) * 16); };
    // The scales of a weight fragment's channels and of the wave's tokens.
    auto read_sw = [&](int slot, int f) {
        if constexpr (Grouped)
            return *reinterpret_cast<const f32x4 *>(ring + slot * STAGE + (BN + BM) * BK +
                                                    ((f * WN + wn) * 16 + quad * 4) * 4);
        else
            return f32x4{};
    };
    auto read_sx = [&](int slot, auto &s) {
        if constexpr (Grouped) {
            const float *q = reinterpret_cast<const float *>(ring + slot * STAGE + (BN + BM) * BK + 1024);
#pragma unroll
            for (int t = 0; t < int(sizeof(s) / sizeof(s[0])); ++t) s[t] = q[(t * WM + wm) * 16 + row16];
        }
    };
    // Products of weight fragment f with the stage's token fragments.
    auto row = [&](auto f_, const i32x8 &a, const f32x4 &aw, const auto &b, const auto &bx) {
        constexpr int f = decltype(f_)::value;
#pragma unroll
        for (int t = 0; t < int(sizeof(b) / sizeof(b[0])); ++t) {
            if constexpr (Grouped) {
                Acc part = Acc{0, 0, 0, 0};
                Mma::run(part, a, b[t]);
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    acc[f][t][r] = __builtin_fmaf(float(part[r]), bx[t] * aw[r], acc[f][t][r]);
            } else {
                Mma::run(acc[f][t], a, b[t]);
            }
        }
    };

    // The rest of the first stages' loads.
    pin();
#pragma unroll
    for (int s = 0; s < S; ++s) {
        aim(s, s);
        static_for<0, XI>(dma_x);
        static_for<0, SI>(dma_s);
    }
    int slot = 0;  // of the stage whose token fragments are in registers
    // Step s of three stages: at its start every read of stage s - 1 has arrived (with a shared
    // ring in every wave), so that stage's slot takes stage s - 1 + S. Weight
    // fragments are read one 16-row block ahead of their MFMAs, the next stage's
    // token fragments and first weight fragment under the last block's, once
    // that stage has landed (with a shared ring for every wave: the barrier).
    auto step = [&](int s, i32x8 &a, f32x4 &aw, const auto &b, const auto &bx, auto &nb, auto &nbx) {
        if (s > 0 && s - 1 + S < count) {
            aim(s - 1 + S, slot == 0 ? S - 1 : slot - 1);
            static_for<0, INSTS>(dma);
        }
        static_for<0, NF - 1>([&](auto f_) {
            const i32x8 an = read_w(slot, decltype(f_)::value + 1);
            const f32x4 anw = read_sw(slot, decltype(f_)::value + 1);
            row(f_, a, aw, b, bx);
            a = an, aw = anw;
            pin();  // (a stage's weight fragments at once do not fit the registers)
        });
        slot = slot + 1 == S ? 0 : slot + 1;
        if (s + 1 < count) {  // stage s + 1, with at most one later one in flight
            if (s == 0) wait_vmcnt<XI + SI>();
            else if (s + 2 < count) wait_vmcnt<INSTS>();
            else wait_vmcnt<0>();
        }
        pin();
        wait_lds_reads();
        if constexpr (NWS > 1) __builtin_amdgcn_s_barrier();
        pin();
        // (After the last stage a slot whose fragments go unused: a conditional
        // read would copy every fragment.)
        read_x(slot, nb);
        read_sx(slot, nbx);
        const i32x8 an = read_w(slot, 0);
        const f32x4 anw = read_sw(slot, 0);
        row(std::integral_constant<int, NF - 1>{}, a, aw, b, bx);
        a = an, aw = anw;
    };
    // Of two stages, refilled in halves: halfway through step s (at a barrier) every
    // wave has read the stage's token rows and the first half of its weight rows, and
    // stage s + 2's take their place; at its end the other half. So a whole stage
    // is in flight at every wait, with 1.5 steps to arrive in. Refilled as a whole,
    // none was (4096 tokens x 4 of 32 experts, 4096 x 2048, 256x256 tiles: INT8 187 -> 170
    // us, FP8 178 -> 160; with three stages of weight rows 174, 165). Stages past the
    // walk's end load as zeros, so that the counts hold.
    constexpr int WL = WI / 2, HALF = NF / 2;
    static_assert(S == 3 || (S == 2 && !Grouped && NWS > 1 && WI % 2 == 0 && NF % 2 == 0), "the steps");
    auto half_steps = [&](int s, i32x8 &a, const auto &b, auto &nb) {
        if (s > 0) {
            aim(s + 1, slot ^ 1);
            static_for<WL, WI>(dma_w);
        }
        static_for<0, NF - 1>([&](auto f_) {
            constexpr int f = decltype(f_)::value;
            if constexpr (f == HALF - 1) {
                wait_vmcnt<INSTS>();  // this stage's second half has landed
                pin();
                wait_lds_reads();
                __builtin_amdgcn_s_barrier();
                pin();
            }
            const i32x8 an = read_w(slot, f + 1);
            if constexpr (f == HALF - 1) {
                aim(s + 2, slot);
                static_for<0, WL>(dma_w);
                static_for<0, XI>(dma_x);
            }
            row(f_, a, f32x4{}, b, 0);
            a = an;
            pin();
        });
        slot ^= 1;
        if (s == 0) wait_vmcnt<WL + XI>();  // stage s + 1's token rows and first half
        else wait_vmcnt<INSTS>();
        pin();
        wait_lds_reads();
        __builtin_amdgcn_s_barrier();
        pin();
        read_x(slot, nb);
        const i32x8 an = read_w(slot, 0);
        row(std::integral_constant<int, NF - 1>{}, a, f32x4{}, b, 0);
        a = an;
    };
    auto any_step = [&](int s, i32x8 &a, f32x4 &aw, const auto &b, const auto &bx, auto &nb, auto &nbx) {
        if constexpr (S == 2) half_steps(s, a, b, nb);
        else step(s, a, aw, b, bx, nb, nbx);
    };
    // All stages for the wave's first L token fragments.
    auto walk = [&](auto live_) {
        constexpr int L = decltype(live_)::value;
        i32x8 a, b0[L], b1[L];
        f32x4 aw;
        float x0[L], x1[L];
        wait_vmcnt<(XI + SI) * (S - 1)>();
        if constexpr (NWS > 1) __builtin_amdgcn_s_barrier();
        pin();
        read_x(0, b0);
        read_sx(0, x0);
        a = read_w(0, 0);
        aw = read_sw(0, 0);
        int s = 0;
        for (; s + 1 < count; s += 2) {
            any_step(s, a, aw, b0, x0, b1, x1);
            any_step(s + 1, a, aw, b1, x1, b0, x0);
        }
        if (s < count) any_step(s, a, aw, b0, x0, b1, x1);
    };
    // The waves along the tokens take the tile's 16-row fragments in turn, so a
    // group's short last tile has fewer in every wave, and only those are
    // multiplied (4096 tokens x 4 of 32 experts, 4096 x 2048, 256x256 tiles: INT8
    // 206 -> 194 us, FP8 192 -> 185).
    const int live = (tile.rows - wm * 16 + 16 * WM - 1) / (16 * WM);
    if (count > 0) {
        if constexpr (MT >= 4) {
            if (live >= 4) walk(std::integral_constant<int, 4>{});
            else if (live == 3) walk(std::integral_constant<int, 3>{});
            else if (live == 2) walk(std::integral_constant<int, 2>{});
            else walk(std::integral_constant<int, 1>{});
        } else if constexpr (MT == 2) {
            if (live >= 2) walk(std::integral_constant<int, 2>{});
            else walk(std::integral_constant<int, 1>{});
        } else {
            walk(std::integral_constant<int, MT>{});
        }
    }
    static_assert(MT == 1 || MT == 2 || MT == 4, "the walks above");
    if (tid < BM) {
        const int to = p.scatter ? to_entry : m_base + tid;
        row_to[tid] = tid < tile.rows && uint32_t(to) < uint32_t(p.slots) ? to : -1;
        row_scale[tid] = row_scale_v;
    }
    if (tid < BN) col_scale[tid] = col_scale_v;
    wait_vmcnt<0>();  // (stages past the walk's end still write zeros)
    wait_lds_reads();
    __syncthreads();

    // Scales and stores. One slice: the 16-bit results go through LDS to whole
    // 16-byte pieces of rows. More: the partial tiles are summed there,
    // ascending slices.
    if constexpr (KS == 1) {
        constexpr int PITCH = BN + 8, kPieces = BN / 8, kPass = 64 * W / kPieces;
        static_assert(64 * W % kPieces == 0, "whole rows per pass");
        uint16_t *tile16 = reinterpret_cast<uint16_t *>(lds);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int ml = (t * WM + wm) * 16 + row16;
            const float scale_x = row_scale[ml];
#pragma unroll
            for (int f = 0; f < NF; ++f) {
                const int nl = (f * WN + wn) * 16 + quad * 4;
                float v[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float s = float(acc[f][t][r]) * scale_x;
                    v[r] = s * col_scale[nl + r];
                }
                *reinterpret_cast<uint2 *>(tile16 + ml * PITCH + nl) =
                    p.out_type == F16 ? uint2{pack2(v[0], v[1], f16_t{}), pack2(v[2], v[3], f16_t{})}
                                      : uint2{pack2(v[0], v[1], bf16_t{}), pack2(v[2], v[3], bf16_t{})};
            }
        }
        __syncthreads();
        const int nl = tid % kPieces * 8;
        const bool whole16 = reinterpret_cast<uintptr_t>(p.y) % 16 == 0;
        if (n_base + nl < N) {
#pragma unroll 4
            for (int ml = tid / kPieces; ml < BM; ml += kPass) {
                const int to = row_to[ml];
                const uint4 v = *reinterpret_cast<const uint4 *>(tile16 + ml * PITCH + nl);
                uint16_t *dst = static_cast<uint16_t *>(p.y) + size_t(max(to, 0)) * N + n_base + nl;
                if (to < 0) continue;
                if (whole16) {
                    *reinterpret_cast<uint4 *>(dst) = v;
                } else {
                    reinterpret_cast<uint2 *>(dst)[0] = uint2{v.x, v.y};
                    reinterpret_cast<uint2 *>(dst)[1] = uint2{v.z, v.w};
                }
            }
        }
    } else {
        constexpr int PITCH = BN + 4;  // 32-bit values per row of a partial tile
        constexpr int kPass = 64 * W / (BN / 4);
        using Red = std::conditional_t<Fmt == I8 && !Grouped, int, float>;
        typedef Red Red4 __attribute__((ext_vector_type(4)));
        Red *red = reinterpret_cast<Red *>(lds);
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int f = 0; f < NF; ++f)
                *reinterpret_cast<Red4 *>(red + (ks * BM + (t * WM + wm) * 16 + row16) * PITCH +
                                          (f * WN + wn) * 16 + quad * 4) = acc[f][t];
        __syncthreads();
        const int nl = tid % (BN / 4) * 4, r0 = tid / (BN / 4);
        if (n_base + nl >= N || r0 >= kPass) return;
        for (int ml = r0; ml < tile.rows; ml += kPass) {
            const int to = row_to[ml];
            if (to < 0) continue;
            Red4 sum = {0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < KS; ++q)
                sum += *reinterpret_cast<const Red4 *>(red + (q * BM + ml) * PITCH + nl);
            float v[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float s = float(sum[r]) * row_scale[ml];
                v[r] = s * col_scale[nl + r];
            }
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p.y) + size_t(to) * N + n_base + nl) =
                p.out_type == F16 ? uint2{pack2(v[0], v[1], f16_t{}), pack2(v[2], v[3], f16_t{})}
                                  : uint2{pack2(v[0], v[1], bf16_t{}), pack2(v[2], v[3], bf16_t{})};
        }
    }
}

template <int Fmt, bool Grouped, int KS, int WN, int WM, int NF, int MT, int S, int EU>
int launch(const ExpertArgs &a, hipStream_t stream) {
    constexpr int W = KS * WN * WM, BN = 16 * NF * WN, BM = 16 * MT * WM;
    constexpr size_t lds = expert_body_bytes(Grouped, KS, S, BN, BM) + (2 * BM + BN) * 4;
    static_assert(lds <= kLdsBytes, "LDS");
    const int tiles_n = (a.N + BN - 1) / BN;
    const int steps = ((a.K + 127) / 128 + KS - 1) / KS;
    hipLaunchKernelGGL((expert_gemm<Fmt, Grouped, KS, WN, WM, NF, MT, S, EU>),
                       dim3(unsigned(expert_row_tiles(a.slots, a.experts, BM) * tiles_n)),
                       dim3(64 * W), lds, stream, a, tiles_n, steps);
    return 0;
}

template <int Fmt, bool Grouped> int launch_any(const ExpertArgs &a, int tile, hipStream_t s) {
#define QLIN_EXPERT_TILE(I, KS, WN, WM, NF, MT, S, EU) \
    case I: return launch<Fmt, Grouped, KS, WN, WM, NF, MT, S, EU>(a, s);
    switch (tile) { QLIN_EXPERT_TILES(QLIN_EXPERT_TILE) }
    if constexpr (!Grouped)
        switch (tile) { QLIN_EXPERT_WIDE_TILES(QLIN_EXPERT_TILE) }
#undef QLIN_EXPERT_TILE
    return -4;
}

}  // namespace

int QLIN_EXPERT_PART(const ExpertArgs &a, int tile, hipStream_t s) {
    return launch_any<QLIN_EXPERT_FMT, QLIN_EXPERT_GROUPED>(a, tile, s);
}
#else
int launch_expert_i8(const ExpertArgs &, int, hipStream_t);
int launch_expert_i8_grouped(const ExpertArgs &, int, hipStream_t);
int launch_expert_fp8(const ExpertArgs &, int, hipStream_t);
int launch_expert_fp8_grouped(const ExpertArgs &, int, hipStream_t);
int launch_expert(const ExpertArgs &a, int tile, hipStream_t s) {
    if (a.fmt == I8) return a.group ? launch_expert_i8_grouped(a, tile, s) : launch_expert_i8(a, tile, s);
    return a.group ? launch_expert_fp8_grouped(a, tile, s) : launch_expert_fp8(a, tile, s);
}
#endif

}  // namespace qlin
