// Rows grouped by the weights they use, for gfx950: the router (top_k experts
// and softmax weights per token), the stable grouping of rows by id, and the
// weighted return of the experts' rows to their tokens.
#include "qlin_internal.hpp"
#include "row_encode.hpp"
#include "row_groups.hpp"

#include <algorithm>

namespace qlin {
namespace {

// ---------------------------------------------------------------- top_k
// Order-preserving key of a logit: larger logit, larger key; 0 for -inf and
// NaN (switched off). -0 and +0 get one key (v + 0 is +0 for both).
__device__ __forceinline__ uint32_t logit_key(float v) {
    if (!(v > -__builtin_inff())) return 0;
    const uint32_t u = __float_as_uint(v + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_logit(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <int Type> __device__ __forceinline__ float load_logit(const void *p, size_t i) {
    if constexpr (Type == F32) return static_cast<const float *>(p)[i];
    else if constexpr (Type == F16) return to_float(static_cast<const uint16_t *>(p)[i], f16_t{});
    else return to_float(static_cast<const uint16_t *>(p)[i], bf16_t{});
}

// f over the lanes' values of an aligned group of L lanes (16 or 64).
template <int L, class V, class F> __device__ __forceinline__ V across(V v, F f) {
    auto other = [&](auto s_) {
        return __builtin_bit_cast(V, lane_xor<decltype(s_)::value>(__builtin_bit_cast(float, v)));
    };
    v = f(v, other(std::integral_constant<int, 1>{}));
    v = f(v, other(std::integral_constant<int, 2>{}));
    v = f(v, other(std::integral_constant<int, 4>{}));
    v = f(v, other(std::integral_constant<int, 8>{}));
    if constexpr (L > 16) {
        v = f(v, other(std::integral_constant<int, 16>{}));
        v = f(v, other(std::integral_constant<int, 32>{}));
    }
    return v;
}

// One token by L lanes of a wave (an aligned group), V logits each: expert
// i * L + l in lane l. Each round takes the largest key left, the lowest expert
// of equals. The low 13 bits of a widened 16-bit logit are zero, so its key's low
// 10 take 1023 - expert and one maximum finds both; fp32 keys need a second pass
// for the expert.
// Bound by the rounds' chains of cross-lane maxima, not by the logits' bytes: 16 lanes for
// up to 128 experts keep a wave's four tokens in one chain (8191 tokens, 8 of 128, bf16:
// 7.5 us with the counting below; 16 tokens, 6 of 64, fp32, sort included: 5.1).
// Choice j ends in lane j (top_k <= 16 <= L): p = e^(v - max), the weights' sum in
// fp32 over the lanes (normalized), or over all logits, per lane first.
// Returns the lane's choice.
template <int Type, int L, int V>
__device__ __forceinline__ int route_token(const RouteArgs &a, int token) {
    constexpr bool kPacked = Type != F32;
    const int l = threadIdx.x % L;
    uint32_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i * L + l;
        const float v = load_logit<Type>(a.logits, size_t(token) * a.ld + min(e, a.experts - 1));
        key[i] = e < a.experts ? logit_key(v) : 0;
        if (kPacked && key[i]) key[i] = (key[i] & ~0x3ffu) | uint32_t(0x3ff - e);
    }
    // The logit of a key as kept.
    auto value = [&](uint32_t k) {
        if constexpr (kPacked) k = k & 0x80000000u ? k & ~0x3ffu : k | 0x3ffu;
        return key_logit(k);
    };
    auto larger = [](uint32_t x, uint32_t y) { return x > y ? x : y; };
    uint32_t mine = 0;
    int expert = -1;
    float peak = 0.f, sum = 0.f;
    for (int j = 0; j < a.top_k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < V; ++i) best = larger(best, key[i]);
        best = across<L>(best, larger);
        if (best == 0) break;  // the same in all L lanes
        if (j == 0) {
            peak = value(best);
            if (!a.normalize) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (key[i]) sum += value(key[i]) == peak ? 1.f : qexp(value(key[i]) - peak);
            }
        }
        int at;
        if constexpr (kPacked) {
            at = 0x3ff - int(best & 0x3ffu);
        } else {
            at = 0x7fffffff;
#pragma unroll
            for (int i = V - 1; i >= 0; --i)
                if (key[i] == best) at = i * L + l;
            at = across<L>(at, [](int x, int y) { return x < y ? x : y; });
        }
        if (l == j) mine = best, expert = at;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * L + l == at) key[i] = 0;
    }
    // (At the maximum itself, +inf too, p is 1; below a maximum of +inf it is 0.)
    const float p = expert < 0 ? 0.f : value(mine) == peak ? 1.f : qexp(value(mine) - peak);
    sum = across<L>(a.normalize ? p : sum, [](float x, float y) { return x + y; });
    if (l < a.top_k) {
        a.ids[size_t(token) * a.top_k + l] = expert;
        a.weights[size_t(token) * a.top_k + l] = expert < 0 ? 0.f : p / sum;
    }
    return expert;
}

static_assert(kMaxGroups == 1024, "an expert's number in 10 bits");
constexpr int kRouteThreads = 256;
template <int Type, int L, int V>
__global__ __launch_bounds__(kRouteThreads) void route_tokens(RouteArgs a) {
    const int token = blockIdx.x * (kRouteThreads / L) + threadIdx.x / L;
    if (token < a.tokens) route_token<Type, L, V>(a, token);
}

// ---------------------------------------------------------------- grouping
// Stable counting sort of ids by group. A wave takes 64 ids at a time in order;
// lanes with the same id find each other with one ballot per id bit, so an
// id's rank is a population count and one lane per distinct id updates the
// wave's counter in LDS: no atomics, the same order every time. One workgroup up to 4096
// ids (57: 3.2 us, its barriers and two passes over the ids); above, the placing launch
// reads every run's counts (65528 ids of 128 groups, 128 runs: 6.3 us).
constexpr int kGroupThreads = 1024, kGroupWaves = kGroupThreads / 64;

// Lanes of the wave with this lane's id (0 for lanes without a valid one).
__device__ __forceinline__ uint64_t same_id(int id, bool valid, int bits) {
    uint64_t m = __ballot(valid);
    for (int b = 0; b < bits; ++b) {
        const uint64_t set = __ballot((id >> b) & 1);
        m &= (id >> b) & 1 ? set : ~set;
    }
    return valid ? m : 0;
}

// Counts of the ids [begin, end) of this workgroup's wave into counts[wave][G].
__device__ __forceinline__ void count_ids(const int *ids, int begin, int end,
                                          int groups, int bits, int *counts) {
    const int lane = threadIdx.x & 63;
    for (int i0 = begin; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const int id = i < end ? ids[i] : -1;
        const bool valid = uint32_t(id) < uint32_t(groups);
        const uint64_t same = same_id(id, valid, bits);
        if (valid && __builtin_ctzll(same) == lane) counts[id] += __builtin_popcountll(same);
        __builtin_amdgcn_wave_barrier();  // the next 64 ids' lanes read it
    }
}
// Slots of the same ids, `next` holding the wave's next slot per group.
__device__ __forceinline__ void place_ids(const GroupArgs &a, int begin, int end, int bits,
                                          int *next) {
    const int lane = threadIdx.x & 63;
    for (int i0 = begin; i0 < end; i0 += 64) {
        const int i = i0 + lane;
        const int id = i < end ? a.ids[i] : -1;
        const bool valid = uint32_t(id) < uint32_t(a.groups);
        const uint64_t same = same_id(id, valid, bits);
        const int rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        const int slot = valid ? next[id] + rank : -1;
        if (i < end) a.slots[i] = slot;
        // (Always within the ids, unless another call writes the same workspace or ids meanwhile.)
        if (uint32_t(slot) < uint32_t(a.count)) a.order[slot] = i;
        if (valid && rank == 0) next[id] = slot + __builtin_popcountll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// Exclusive prefix sum over the workgroup's threads (one value each).
__device__ __forceinline__ int block_scan(int v, int *shared) {
    const int upto = wave_scan(v);
    if ((threadIdx.x & 63) == 63) shared[threadIdx.x >> 6] = upto;
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) before += w < int(threadIdx.x >> 6) ? shared[w] : 0;
    __syncthreads();
    return before + upto - v;
}

// Per-wave counts in LDS [kGroupWaves][groups] to each wave's first slot, the
// group's first slot being `base` of thread g. Thread g handles group g.
__device__ __forceinline__ void counts_to_slots(int *counts, int groups, int base) {
    const int g = threadIdx.x;
    if (g >= groups) return;
#pragma unroll
    for (int w = 0; w < kGroupWaves; ++w) {
        const int c = counts[w * groups + g];
        counts[w * groups + g] = base;
        base += c;
    }
}

// All ids in one workgroup.
__device__ __forceinline__ void group_in_one(const GroupArgs &a, int bits, int *counts,
                                             int *shared) {
    const int wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kGroupWaves * a.groups; i += kGroupThreads) counts[i] = 0;
    __syncthreads();
    const int each = (a.count + kGroupThreads - 1) / kGroupThreads * 64;  // ids per wave
    const int begin = min(wave * each, a.count), end = min(begin + each, a.count);
    count_ids(a.ids, begin, end, a.groups, bits, counts + wave * a.groups);
    __syncthreads();
    int total = 0;
    if (int(threadIdx.x) < a.groups)
#pragma unroll
        for (int w = 0; w < kGroupWaves; ++w) total += counts[w * a.groups + threadIdx.x];
    const int base = block_scan(total, shared);
    if (int(threadIdx.x) < a.groups) {
        a.offsets[threadIdx.x] = base;
        if (int(threadIdx.x) == a.groups - 1) a.offsets[a.groups] = shared[0] = base + total;
    }
    counts_to_slots(counts, a.groups, base);
    __syncthreads();
    for (int i = shared[0] + threadIdx.x; i < a.count; i += kGroupThreads) a.order[i] = -1;
    place_ids(a, begin, end, bits, counts + wave * a.groups);
}

__global__ __launch_bounds__(kGroupThreads) void group_one(GroupArgs a, int bits) {
    extern __shared__ int counts[];
    __shared__ int shared[kGroupWaves];
    group_in_one(a, bits, counts, shared);
}

// Many ids: workgroup b counts its run of `each` ids into table[b][groups] ...
__global__ __launch_bounds__(kGroupThreads) void group_count(GroupArgs a, int each) {
    __shared__ int counts[kMaxGroups];
    if (int(threadIdx.x) < a.groups) counts[threadIdx.x] = 0;
    __syncthreads();
    const int first = int(blockIdx.x) * each, end = min(first + each, a.count);
    for (int i = first + threadIdx.x; i < end; i += kGroupThreads) {
        const int id = a.ids[i];
        if (uint32_t(id) < uint32_t(a.groups)) atomicAdd(counts + id, 1);  // (sums of ones: any order)
    }
    __syncthreads();
    int *table = static_cast<int *>(a.workspace) + size_t(blockIdx.x) * a.groups;
    if (int(threadIdx.x) < a.groups) table[threadIdx.x] = counts[threadIdx.x];
}
// ... or the router does so for the tokens that it routes ...
template <int Type, int L, int V>
__global__ __launch_bounds__(kGroupThreads) void route_count(RouteArgs r, GroupArgs a) {
    __shared__ int counts[kMaxGroups];
    if (int(threadIdx.x) < a.groups) counts[threadIdx.x] = 0;
    __syncthreads();
    const int token = blockIdx.x * (kGroupThreads / L) + threadIdx.x / L;
    if (token < r.tokens) {
        const int expert = route_token<Type, L, V>(r, token);
        if (int(threadIdx.x % L) < r.top_k && expert >= 0) atomicAdd(counts + expert, 1);
    }
    __syncthreads();
    int *table = static_cast<int *>(a.workspace) + size_t(blockIdx.x) * a.groups;
    if (int(threadIdx.x) < a.groups) table[threadIdx.x] = counts[threadIdx.x];
}
// ... and the ids are placed after the earlier groups and the earlier workgroups' ids.
__global__ __launch_bounds__(kGroupThreads) void group_place(GroupArgs a, int bits, int each) {
    extern __shared__ int counts[];  // [kGroupWaves][groups]
    __shared__ int shared[kGroupWaves], all[kGroupThreads], earlier[kGroupThreads];
    const int wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < kGroupWaves * a.groups; i += kGroupThreads) counts[i] = 0;
    // Column sums of the table, its rows dealt to as many threads a group as there
    // are: all rows' and those of the earlier workgroups.
    const int *table = static_cast<const int *>(a.workspace);
    const int parts = kGroupThreads / a.groups, part = int(threadIdx.x) / a.groups;
    int total = 0, before = 0;
    if (part < parts) {
        const int g = int(threadIdx.x) % a.groups;
#pragma unroll 8
        for (int b = part; b < int(gridDim.x); b += parts) {
            const int c = table[size_t(b) * a.groups + g];
            before += b < int(blockIdx.x) ? c : 0;
            total += c;
        }
    }
    all[threadIdx.x] = total, earlier[threadIdx.x] = before;
    __syncthreads();
    const int first = int(blockIdx.x) * each, share = (each + kGroupThreads - 1) / kGroupThreads * 64;
    const int past = min(first + each, a.count);
    const int begin = min(first + wave * share, past), end = min(begin + share, past);
    count_ids(a.ids, begin, end, a.groups, bits, counts + wave * a.groups);
    total = before = 0;
    if (int(threadIdx.x) < a.groups)
        for (int q = 0; q < parts; ++q)
            total += all[q * a.groups + threadIdx.x], before += earlier[q * a.groups + threadIdx.x];
    const int base = block_scan(total, shared);
    if (int(threadIdx.x) < a.groups) {
        if (blockIdx.x == 0) a.offsets[threadIdx.x] = base;
        if (int(threadIdx.x) == a.groups - 1) {
            shared[0] = base + total;
            if (blockIdx.x == 0) a.offsets[a.groups] = base + total;
        }
    }
    __syncthreads();
    counts_to_slots(counts, a.groups, base + before);
    __syncthreads();
    for (int i = max(shared[0], first) + int(threadIdx.x); i < past; i += kGroupThreads) a.order[i] = -1;
    place_ids(a, begin, end, bits, counts + wave * a.groups);
}

// A decode step's router: every token and the grouping in one workgroup.
template <int Type, int L, int V>
__global__ __launch_bounds__(kGroupThreads) void route_one(RouteArgs r, GroupArgs a, int bits) {
    extern __shared__ int counts[];
    __shared__ int shared[kGroupWaves];
    for (int token = threadIdx.x / L; token < r.tokens; token += kGroupThreads / L)
        route_token<Type, L, V>(r, token);
    __threadfence_block();
    __syncthreads();
    group_in_one(a, bits, counts, shared);
}

constexpr int kOneGroup = 4096;  // ids that one workgroup sorts
int id_bits(int groups) {
    int bits = 0;
    while ((1 << bits) < groups) ++bits;
    return bits;
}
constexpr int kMaxRuns = 256;  // rows of the table, which every workgroup reads
int group_run(int count) { return int((long(count) + kGroupThreads * 64 - 1) / (kGroupThreads * 64)) * kGroupThreads; }
void launch_place(const GroupArgs &a, int run, hipStream_t s) {
    hipLaunchKernelGGL(group_place, dim3(unsigned((long(a.count) + run - 1) / run)), dim3(kGroupThreads),
                       size_t(kGroupWaves) * a.groups * 4, s, a, id_bits(a.groups), run);
}

template <int Type, int L, int V>
void launch_route_as(const RouteArgs &r, const GroupArgs &g, hipStream_t s) {
    constexpr int kTokens = kGroupThreads / L;
    if (r.tokens <= kTokens && g.count <= kOneGroup) {
        hipLaunchKernelGGL((route_one<Type, L, V>), dim3(1), dim3(kGroupThreads),
                           size_t(kGroupWaves) * g.groups * 4, s, r, g, id_bits(g.groups));
        return;
    }
    // Above 4096 choices the router counts them for the grouping (8191 tokens, 8 of 128:
    // 19.2 -> 17.0 us), while its workgroups are no more than the table's rows.
    const int blocks = (r.tokens + kTokens - 1) / kTokens;
    if (g.count > kOneGroup && blocks <= kMaxRuns) {
        hipLaunchKernelGGL((route_count<Type, L, V>), dim3(unsigned(blocks)), dim3(kGroupThreads), 0, s, r, g);
        launch_place(g, kTokens * r.top_k, s);
        return;
    }
    constexpr int each = kRouteThreads / L;
    hipLaunchKernelGGL((route_tokens<Type, L, V>), dim3(unsigned((r.tokens + each - 1) / each)),
                       dim3(kRouteThreads), 0, s, r);
    launch_group_rows(g, s);
}

template <int Type> void launch_route_type(const RouteArgs &r, const GroupArgs &g, hipStream_t s) {
    if (r.experts <= 16) launch_route_as<Type, 16, 1>(r, g, s);
    else if (r.experts <= 64) launch_route_as<Type, 16, 4>(r, g, s);
    else if (r.experts <= 128) launch_route_as<Type, 16, 8>(r, g, s);
    else if (r.experts <= 256) launch_route_as<Type, 64, 4>(r, g, s);
    else launch_route_as<Type, 64, 16>(r, g, s);
}

// ---------------------------------------------------------------- combine
// out[t] = s16(sum_j weights[t, j] * h[slots[t, j]] + base[t]), fp32, ascending
// j; rows without a slot (or past h) are not read. A workgroup takes 2048 columns of a
// token, a thread eight: bound by HBM (4096 tokens, 8 rows of 2048 each and a base: 33.9
// us, 4.9 TB/s).
template <class T, bool Vec>
__global__ __launch_bounds__(kThreads) void combine_rows(CombineArgs a, int tiles) {
    const int token = blockIdx.x / tiles;
    const int column = (int(blockIdx.x % tiles) * kThreads + int(threadIdx.x)) * 8;
    if (column >= a.N) return;
    const int *slots = a.slots + size_t(token) * a.top_k;
    const float *weights = a.weights ? a.weights + size_t(token) * a.top_k : nullptr;
    const uint16_t *h = static_cast<const uint16_t *>(a.h);
    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j = 0; j < a.top_k; ++j) {
        const int slot = slots[j];
        if (uint32_t(slot) >= uint32_t(a.h_rows)) continue;
        const float wt = weights ? weights[j] : 1.f;
        float u[8];
        load8<T, Vec>(h + size_t(slot) * a.N, column, a.N, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __builtin_fmaf(wt, u[i], v[i]);
    }
    if (a.base) {
        float u[8];
        load8<T, Vec>(static_cast<const uint16_t *>(a.base) + size_t(token) * a.N, column, a.N, u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += u[i];
    }
    store16x8<T, Vec>(static_cast<uint16_t *>(a.out) + size_t(token) * a.N, column, a.N, v);
}

}  // namespace

size_t group_workspace_bytes(int count, int groups) {
    if (count <= kOneGroup) return 0;
    static_assert(kMaxRuns >= 64, "group_run's rows");
    return size_t(kMaxRuns) * groups * 4;
}

void launch_group_rows(const GroupArgs &a, hipStream_t s) {
    if (a.count <= kOneGroup) {
        hipLaunchKernelGGL(group_one, dim3(1), dim3(kGroupThreads), size_t(kGroupWaves) * a.groups * 4, s, a,
                           id_bits(a.groups));
        return;
    }
    const int run = group_run(a.count);
    hipLaunchKernelGGL(group_count, dim3(unsigned((long(a.count) + run - 1) / run)), dim3(kGroupThreads), 0, s,
                       a, run);
    launch_place(a, run, s);
}

void launch_route(const RouteArgs &r, const GroupArgs &g, hipStream_t s) {
    if (r.type == F32) launch_route_type<F32>(r, g, s);
    else if (r.type == F16) launch_route_type<F16>(r, g, s);
    else launch_route_type<BF16>(r, g, s);
}

void launch_combine(const CombineArgs &a, hipStream_t s) {
    auto at16 = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool vec = a.N % 8 == 0 && at16(a.h) && at16(a.out) && at16(a.base);
    const int tiles = (a.N + kChunk - 1) / kChunk;
    const dim3 grid(unsigned(long(a.tokens) * tiles));
#define QLIN_COMBINE(T, V) \
    hipLaunchKernelGGL((combine_rows<T, V>), grid, dim3(kThreads), 0, s, a, tiles)
    if (a.type == F16) {
        if (vec) QLIN_COMBINE(f16_t, true);
        else QLIN_COMBINE(f16_t, false);
    } else {
        if (vec) QLIN_COMBINE(bf16_t, true);
        else QLIN_COMBINE(bf16_t, false);
    }
#undef QLIN_COMBINE
}

}  // namespace qlin
