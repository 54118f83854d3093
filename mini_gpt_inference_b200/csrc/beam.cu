// A beam search's step on the device: which continuations go on (select), and the caches of the rows that do not, handed
// over to the rows that do (reorder).
//
// Select.  A group has I rows of logits (its beams) and a score for each, the sum of its tokens' log probabilities.  A
// candidate (b, t) is worth  v = score_b + logit_bt - L_b,  L_b = log sum_t exp logit_bt, and is ranked by v / len^a, len the
// tokens of the continuation.  The B best go on.  Equal ranks go to the lower row; within a row the order is that of the
// logits, equal ones by the lower id, so a row's B largest logits are all that a row can contribute, whatever L_b is:
//
//   rows kernel    one pass over the logits: every lane of a CTA keeps the maximum and sum of its own (for L_b).  The B best
//                  logits of the CTA's piece lie in the lanes with the B largest maxima; those lanes' logits are looked at again.
//                  (logit, id) pairs are 64-bit keys, the logit's bits in an order that unsigned numbers have, then the id
//                  from above: all keys differ, so ties need no care.  Lists are sorted over a warp's lanes and joined by
//                  bitonic merges.  (Every warp keeping the B best of its piece as it reads: 768 instructions for 512 logits
//                  of 50,257 and B = 16, and bound by them: 85 us for 64 x 16 rows.)
//   choice kernel  one CTA a group: the rows' lists and sums joined, values in 64 bits, and the candidates in front of each
//                  counted.
//
// A beam that goes on stays in its row: its best continuation takes the row, its others take, in order of rank, the rows
// whose beams do not go on.  So only those rows' caches change hands, a row that is read is never written (reorder needs
// no second buffer), and a search whose beams are stable copies nothing.  `ranks` tells the order.
//
// A logit that is no number counts as minus infinity, and so does a value that is none (a row with an infinite logit, or with
// none above minus infinity).  A beam that has ended has one candidate, itself.
#include <math.h>

#include "common.cuh"

MG_GUARD_DECLARE(beam)

namespace {

typedef unsigned long long u64;

constexpr int MAX_BEAMS = 32;
constexpr int ROW_THREADS = 256, ROW_WARPS = ROW_THREADS / 32;
constexpr int BATCH = 512;              // logits that a warp takes at a time: 16 a lane

// Bits of a number in the order of unsigned integers (minus zero as zero; 0 is below every number's).
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t o) { return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ u64 order_of(double x) {
    const u64 b = (u64)__double_as_longlong(x + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 1ull << 63);
}

__device__ __forceinline__ u64 key_of(float x, int id) { return ((u64)order_of(x) << 32) | (uint32_t)~(uint32_t)id; }

__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }
__device__ __forceinline__ u64 min64(u64 a, u64 b) { return a < b ? a : b; }

// The 32 largest of two lists, sorted downwards over the lanes.
__device__ __forceinline__ u64 merge_lists(u64 a, u64 b, int lane) {
    u64 c = max64(a, __shfl_xor_sync(0xffffffffu, b, 31));          // first half of a bitonic sequence
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 other = __shfl_xor_sync(0xffffffffu, c, o);
        c = (lane & o) ? min64(c, other) : max64(c, other);
    }
    return c;
}

// The 32 largest of two lists of numbers, and the lanes' numbers, sorted downwards over the lanes.
__device__ __forceinline__ uint32_t merge_lists(uint32_t a, uint32_t b, int lane) {
    uint32_t c = max(a, __shfl_xor_sync(0xffffffffu, b, 31));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const uint32_t other = __shfl_xor_sync(0xffffffffu, c, o);
        c = (lane & o) ? min(c, other) : max(c, other);
    }
    return c;
}
__device__ __forceinline__ uint32_t sort_lanes(uint32_t v, int lane) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int o = k >> 1; o > 0; o >>= 1) {
            const uint32_t other = __shfl_xor_sync(0xffffffffu, v, o);
            v = ((lane & k) == 0) == ((lane & o) == 0) ? max(v, other) : min(v, other);
        }
    return v;
}

// The 32 largest keys of the CTA's warps, sorted downwards over the lanes of warp 0, from lists that are so in every warp.
template <typename T>
__device__ __forceinline__ T merge_warps(T list, T (&meet)[ROW_WARPS][32], int warp, int lane) {
    meet[warp][lane] = list;
#pragma unroll
    for (int half = ROW_WARPS / 2; half > 0; half >>= 1) {
        __syncthreads();
        if (warp < half) {
            list = merge_lists(list, meet[warp + half][lane], lane);
            meet[warp][lane] = list;
        }
    }
    return list;
}

__global__ void __launch_bounds__(ROW_THREADS)
beam_rows_kernel(const float* __restrict__ logits, const int* __restrict__ ended, u64* __restrict__ lists, float* __restrict__ sums,
                 int vocab, int limit, int beams, int chunk) {
    __shared__ u64 meet[ROW_WARPS][32];
    __shared__ uint32_t meet_order[ROW_WARPS][32], owners[ROW_WARPS][2], bound_s;
    __shared__ float meet_max[ROW_WARPS], meet_sum[ROW_WARPS];
    const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_wait();
    pdl_trigger();
    if (ended != nullptr && ended[row] != 0) return;       // its one candidate is itself
    const float* const base = logits + (size_t)row * vocab;
    // ids are counted from the 16-byte boundary at or in front of the row's first logit
    const int lead = (int)(((uintptr_t)base >> 2) & 3);
    const int begin = (blockIdx.x * ROW_WARPS + warp) * chunk, end = min(limit + lead, begin + chunk);
    const float log2e = 1.4426950408889634f;
    // One pass for the sums and every lane's largest logit (16 a batch and lane, four neighbours at a time; what is not there, or
    // no number, is minus infinity).
    auto quad = [&](int at, float (&x)[4]) {
        if (at >= lead && at + 4 <= end) {
            const float4 v = *reinterpret_cast<const float4*>(base + (at - lead));
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = (at + i >= lead && at + i < end) ? base[at + i - lead] : -INFINITY;
        }
    };
    float top = -INFINITY, sum = 0.f, next_x[4][4];
    if (begin < end)
#pragma unroll
        for (int q = 0; q < 4; ++q) quad(begin + q * 128 + lane * 4, next_x[q]);
    for (int b0 = begin; b0 < end; b0 += BATCH) {
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = fmaxf(next_x[e >> 2][e & 3], -INFINITY);
        if (b0 + BATCH < end)                               // on its way while these are looked at
#pragma unroll
            for (int q = 0; q < 4; ++q) quad(b0 + BATCH + q * 128 + lane * 4, next_x[q]);
        float high = x[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) high = fmaxf(high, x[e]);
        if (high > top) {                                   // the sum is relative to the largest so far
            sum *= exp2f((top - high) * log2e);
            top = high;
        }
        // (first the difference, then log2 e: what is rounded does not grow with the logits, and the largest one counts as 1)
        const float base = top == -INFINITY ? 0.f : top;
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 16; ++e) part[e & 3] += exp2_approx((x[e] - base) * log2e);
        sum += (part[0] + part[1]) + (part[2] + part[3]);
    }
    const float warp_top = warp_max(top);
    sum = warp_sum(warp_top == -INFINITY ? 0.f : sum * exp2f((top - warp_top) * log2e));
    if (lane == 0) { meet_max[warp] = warp_top; meet_sum[warp] = sum; }
    // The CTA's 256 lanes have `beams` logits not below the beams-th largest of their maxima: what is as good lies in the lanes
    // whose maximum is, and their logits are looked at once more, a lane's by a warp.  (Lanes without logits count as minus
    // infinity here and add nothing there; where fewer than `beams` lanes have some, that is the bound.)  Equal logits go by their
    // ids, which rise with the warps: once `beams` lanes reach the bound, later warps' lanes have to pass it.  (64 x 16
    // rows of 50,257 equal logits, or of all but three minus infinity, together with the launches: 104 us, 212 without that.)
    const uint32_t maxima = merge_warps(sort_lanes(order_of(top), lane), meet_order, warp, lane);
    if (warp == 0) {
        const uint32_t bound = __shfl_sync(0xffffffffu, maxima, beams - 1);
        if (lane == 0) bound_s = bound;
    }
    __syncthreads();
    const float bound = number_of(bound_s);
    const uint32_t good = __ballot_sync(0xffffffffu, begin < end && top >= bound), better = __ballot_sync(0xffffffffu, top > bound);
    if (lane == 0) { owners[warp][0] = good; owners[warp][1] = better; }
    __syncthreads();
    u64 list = 0, least = 0;                                // lane i: the warp's i-th best; its beams-th best
    int turn = 0, reach = 0;                                // lanes taken; lanes of the warps so far that reach the bound
    for (int w = 0; w < ROW_WARPS; ++w) {
        const int first = (blockIdx.x * ROW_WARPS + w) * chunk, last = min(limit + lead, first + chunk);
        uint32_t left = owners[w][reach >= beams];
        reach += __popc(owners[w][0]);
        for (; left; left &= left - 1, ++turn) {
            if (turn % ROW_WARPS != warp) continue;
            const int column = first + (__ffs(left) - 1) * 4;
            for (int j = column + lane * 128; __any_sync(0xffffffffu, j < last); j += 32 * 128) {
                float x[4];
                if (j >= lead && j + 4 <= last) {
                    const float4 v = *reinterpret_cast<const float4*>(base + (j - lead));
                    x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = (j + i >= lead && j + i < last) ? base[j + i - lead] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = fmaxf(x[i], -INFINITY);
                    const u64 mine = x[i] >= bound && j + i >= lead && j + i < last ? key_of(x[i], j + i - lead) : 0;
                    uint32_t todo = __ballot_sync(0xffffffffu, mine > least);
                    while (todo) {
                        const u64 next = __shfl_sync(0xffffffffu, mine, __ffs(todo) - 1);
                        todo &= todo - 1;
                        if (next <= least) continue;        // (the list has grown since the ballot)
                        const int place = __popc(__ballot_sync(0xffffffffu, list > next));
                        const u64 up = __shfl_up_sync(0xffffffffu, list, 1);
                        list = lane < place ? list : lane == place ? next : up;
                        least = __shfl_sync(0xffffffffu, list, beams - 1);
                    }
                }
            }
        }
    }
    list = merge_warps(list, meet, warp, lane);
    if (warp == 0) {
        const size_t at = (size_t)row * gridDim.x + blockIdx.x;
        if (lane < beams) lists[at * beams + lane] = list;
        const float m = lane < ROW_WARPS ? meet_max[lane] : -INFINITY;
        const float all = warp_max(m);
        const float s = warp_sum(lane < ROW_WARPS && all != -INFINITY ? meet_sum[lane] * exp2f((m - all) * log2e) : 0.f);
        if (lane == 0) *reinterpret_cast<float2*>(sums + at * 2) = make_float2(all, s);
    }
}

struct ChoiceArgs {
    const u64* lists;
    const float* sums;
    const float* scores;
    const int* ended;
    const int* lengths;
    int* tokens;
    int* parents;
    float* scores_out;
    int* ranks;
    int* ended_out;
    int* lengths_out;
    int in_beams, beams, parts, end_token;
    double penalty;
};

__global__ void __launch_bounds__(1024) beam_choice_kernel(const __grid_constant__ ChoiceArgs a) {
    __shared__ u64 meet[32][32];                         // lists of the warps, then the candidates' ranks [row][order]
    __shared__ double value[32][32], row_total[32], row_weight[32];
    __shared__ int token[32][32], rank[32][32], row_length[32], row_over[32], choice[32];
    const int group = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    const int per_row = warps / a.in_beams;               // warps that share a row's lists, a power of two
    const int b = warp / per_row, share = warp - b * per_row;
    const int row = group * a.in_beams + b;
    // (the row's first warp ends up with its list; the last one works out what the logits are measured against meanwhile)
    const bool leads = share == 0, sums_up = share == per_row - 1;
    pdl_wait();
    pdl_trigger();
    const bool over = a.ended != nullptr && a.ended[row] != 0;
    const double before = (double)a.scores[row];
    const int length = (a.lengths != nullptr ? max(0, a.lengths[row]) : 0) + (over ? 0 : 1);
    u64 list = 0;
    if (!over)
        for (int i = share; i < a.parts; i += per_row)
            list = merge_lists(list, lane < a.beams ? a.lists[((size_t)row * a.parts + i) * a.beams + lane] : 0, lane);
    if (sums_up) {
        double total = 0.0;
        if (!over) {
            // the sums, relative to the largest maximum
            float2 ms = lane < a.parts ? *reinterpret_cast<const float2*>(a.sums + ((size_t)row * a.parts + lane) * 2) : make_float2(-INFINITY, 0.f);
            for (int i = lane + 32; i < a.parts; i += 32) {
                const float2 more = *reinterpret_cast<const float2*>(a.sums + ((size_t)row * a.parts + i) * 2);
                const float high = fmaxf(ms.x, more.x);
                if (high != -INFINITY)
                    ms.y = ms.y * exp2f((ms.x - high) * 1.4426950408889634f) + more.y * exp2f((more.x - high) * 1.4426950408889634f);
                ms.x = high;
            }
            const float m = warp_max(ms.x);
            double s = ms.x != -INFINITY ? (double)ms.y * (double)exp2f((ms.x - m) * 1.4426950408889634f) : 0.0;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            total = (double)m + log(s);
        }
        if (lane == 0) {
            row_total[b] = total;
            row_weight[b] = a.penalty == 0.0 ? 1.0 : a.penalty == 1.0 ? (double)max(1, length) : pow((double)max(1, length), a.penalty);
            row_length[b] = length;
            row_over[b] = over;
        }
    }
    for (int half = per_row >> 1; half > 0; half >>= 1) {
        if (share >= half && share < 2 * half) meet[warp][lane] = list;
        __syncthreads();
        if (share < half) list = merge_lists(list, meet[warp + half][lane], lane);
        __syncthreads();
    }
    if (per_row == 1) __syncwarp();
    if (leads && lane < a.beams) {
        double v = over ? (lane == 0 ? before : -INFINITY) : before + ((double)number_of((uint32_t)(list >> 32)) - row_total[b]);
        if (!(v == v)) v = -INFINITY;
        double weighed = v / row_weight[b];
        if (!(weighed == weighed)) weighed = -INFINITY;
        value[b][lane] = v;
        token[b][lane] = over ? a.end_token : (int)~(uint32_t)list;
        meet[b][lane] = order_of(weighed);
        rank[b][lane] = lane;
    }
    __syncthreads();
    // A candidate's rank is its place in its own row and, in each other row, the number of candidates in front of it (equal ones of
    // a lower row are), by bisection: a thread a candidate and other row.
    const int candidates = a.in_beams * a.beams;
    for (int x = threadIdx.x; x < candidates * a.in_beams; x += blockDim.x) {
        const int other = x / candidates, c = x - other * candidates, r = c / a.beams, order = c - r * a.beams;
        const u64 mine = meet[r][order];
        int lo = 0, hi = other == r ? 0 : a.beams;        // candidates of `other` that come first: [0, lo)
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            const u64 theirs = meet[other][mid];
            if (theirs > mine || (theirs == mine && other < r)) lo = mid + 1; else hi = mid;
        }
        if (lo > 0) atomicAdd(&rank[r][order], lo);
    }
    __syncthreads();
    if (leads && lane < a.beams && rank[b][lane] < a.beams) choice[rank[b][lane]] = b * 32 + lane;
    __syncthreads();
    if (warp != 0) return;
    // rows: the best continuation of a beam takes its row, the others the rows that are left, in order
    const bool chosen = lane < a.beams;
    const int from = chosen ? choice[lane] >> 5 : 0, order = chosen ? choice[lane] & 31 : 0;
    const uint32_t same = __match_any_sync(0xffffffffu, chosen ? from : 32 + lane);
    const bool stays = chosen && (same & ((1u << lane) - 1u)) == 0u;
    const uint32_t taken = __reduce_or_sync(0xffffffffu, stays ? 1u << from : 0u);
    const uint32_t moved = __ballot_sync(0xffffffffu, chosen && !stays);
    int to = from;
    if (chosen && !stays) {
        uint32_t free = ~taken;
        for (int i = __popc(moved & ((1u << lane) - 1u)); i > 0; --i) free &= free - 1u;
        to = __ffs(free) - 1;
    }
    if (chosen) {
        const int out_row = group * a.beams + to, t = token[from][order];
        a.tokens[out_row] = t;
        a.parents[out_row] = group * a.beams + from;
        a.scores_out[out_row] = (float)value[from][order];
        a.ranks[out_row] = lane;
        if (a.ended_out != nullptr) a.ended_out[out_row] = row_over[from] != 0 || t == a.end_token;
        if (a.lengths_out != nullptr) a.lengths_out[out_row] = row_length[from];
    }
}

// Logits of one warp's piece, in batches: as many warps as keep the GPU busy, but not more lists than that needs.
int chunk_of(int rows, int limit) {
    const long long warps = 148 * 32;                     // half of what the GPU holds at once
    long long batches = ((long long)rows * limit + BATCH * warps - 1) / (BATCH * warps);
    if (batches < 1) batches = 1;
    if (batches > 8) batches = 8;
    const int ctas = ceil_div(limit + 3, (int)batches * BATCH * ROW_WARPS);
    return ceil_div(ceil_div(limit + 3, ctas * ROW_WARPS), BATCH) * BATCH;      // even pieces
}
int parts_of(int rows, int limit) { return ceil_div(limit + 3, chunk_of(rows, limit) * ROW_WARPS); }

// ---- caches of rows that do not go on -----------------------------------------------------------------------------
constexpr int MAX_PAGED = 8, MAX_STATES = 48;

struct Paged {
    int* table;              // [rows][width]
    char* k;                 // [layer][page][kv head][token][feature]
    char* v;                 // the same, or null
    long long k_layer, v_layer;                // bytes of a layer
    int k_token, v_token;                      // bytes of a token's features in a head
    int width, page_tokens, num_pages, n_kv_head, layers, unit;      // unit: bytes that are moved at a time
};
struct State {
    char* data;              // [slot][bytes]
    long long bytes;
    int unit, slots;
};
struct ReorderArgs {
    const int* parents;
    const int* lengths;
    const int* slots;
    int rows, n_paged, n_states;
    Paged paged[MAX_PAGED];
    State state[MAX_STATES];
};

template <typename V>
__device__ __forceinline__ void move_run(char* to, const char* of, long long bytes, long long at, long long step) {
    // several pieces on their way before the first is stored
    constexpr int U = sizeof(V) == 16 ? 4 : 8;
    const long long n = bytes / (long long)sizeof(V);
    for (long long i = at; i < n; i += U * step) {
        V v[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (i + k * step < n) v[k] = reinterpret_cast<const V*>(of)[i + k * step];
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (i + k * step < n) reinterpret_cast<V*>(to)[i + k * step] = v[k];
    }
}

__device__ __forceinline__ void move_bytes(char* to, const char* of, long long bytes, int unit, long long at, long long step) {
    if (unit == 16) move_run<uint4>(to, of, bytes, at, step);
    else if (unit == 8) move_run<uint2>(to, of, bytes, at, step);
    else if (unit == 4) move_run<uint32_t>(to, of, bytes, at, step);
    else if (unit == 2) move_run<uint16_t>(to, of, bytes, at, step);
    else move_run<uint8_t>(to, of, bytes, at, step);
}

// CTA (piece, row, tensor): rows whose parent is another row take over what is the parent's.
__global__ void __launch_bounds__(256, 4) beam_reorder_kernel(const __grid_constant__ ReorderArgs a) {
    pdl_trigger();
    pdl_wait();
    const int row = blockIdx.y;
    const int parent = a.parents[row], which = blockIdx.z;
    if (parent == row || parent < 0 || parent >= a.rows) return;
    const int grand = a.parents[parent], length = which < a.n_paged ? a.lengths[parent] : 0;
    if (grand != parent) return;                          // (the parent takes over another row itself: see above)
    if (which < a.n_paged) {
        const Paged& p = a.paged[which];
        const int full = length / p.page_tokens, used = length - full * p.page_tokens;
        int* const mine = p.table + (size_t)row * p.width;
        const int* const theirs = p.table + (size_t)parent * p.width;
        if (length <= 0) return;
        for (int c = blockIdx.x * blockDim.x + threadIdx.x; c < min(full, p.width); c += gridDim.x * blockDim.x) mine[c] = theirs[c];
        if (used == 0 || full >= p.width) return;
        const int to = mine[full], of = theirs[full];
        if (to < 0 || of < 0 || to >= p.num_pages || of >= p.num_pages || to == of) return;
        // runs of `used` tokens, one per layer and head: a warp each
        const int warp = (blockIdx.x * blockDim.x + threadIdx.x) >> 5, warps = (gridDim.x * blockDim.x) >> 5, lane = threadIdx.x & 31;
        const int runs = p.layers * p.n_kv_head * (p.v != nullptr ? 2 : 1);
        for (int r = warp; r < runs; r += warps) {
            const bool is_v = r >= p.layers * p.n_kv_head;
            const int i = is_v ? r - p.layers * p.n_kv_head : r, layer = i / p.n_kv_head, head = i - layer * p.n_kv_head;
            const long long token = is_v ? p.v_token : p.k_token;
            char* const base = (is_v ? p.v : p.k) + layer * (is_v ? p.v_layer : p.k_layer);
            move_bytes(base + ((long long)to * p.n_kv_head + head) * p.page_tokens * token,
                       base + ((long long)of * p.n_kv_head + head) * p.page_tokens * token, used * token, p.unit, lane, 32);
        }
    } else {
        const State& s = a.state[which - a.n_paged];
        const int to = a.slots[row], of = a.slots[parent];
        if (to < 0 || of < 0 || to >= s.slots || of >= s.slots || to == of) return;
        move_bytes(s.data + to * s.bytes, s.data + of * s.bytes, s.bytes, s.unit, (long long)blockIdx.x * blockDim.x + threadIdx.x,
                   (long long)gridDim.x * blockDim.x);
    }
}

int unit_of(uintptr_t bits) { return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1; }

}  // namespace

// Bytes of scratch for mg_beam_select (16-byte aligned).
MG_API long long mg_beam_select_scratch_bytes(int groups, int in_beams, int beams, int limit) {
    if (groups <= 0 || in_beams <= 0 || beams <= 0 || limit <= 0) return 0;
    return (long long)groups * in_beams * parts_of(groups * in_beams, limit) * (8ll * beams + 8);
}

// logits [groups * in_beams, vocab] 32-bit; scores [groups * in_beams]; ended, lengths [groups * in_beams] ints or null; outputs
// [groups * beams].  Ids at or above `limit` do not exist (they have no part in the sums either).  end_token: what ended
// beams go on with, and what ends a beam (-1: none).  lengths_out may be null where lengths is; ended_out without ended
// given starts from beams that have not ended.  scratch: mg_beam_select_scratch_bytes(), used by no other launch meanwhile.
MG_API int mg_beam_select(const float* logits, const float* scores, const int* ended, const int* lengths, int groups, int in_beams,
                          int beams, int vocab, int limit, int end_token, double penalty, int* tokens, int* parents,
                          float* scores_out, int* ranks, int* ended_out, int* lengths_out, void* scratch, void* stream) {
    if (groups == 0) return MG_OK;
    MG_REQUIRE(groups > 0 && in_beams > 0 && in_beams <= beams && beams <= MAX_BEAMS, "beam_select: bad numbers of beams");
    MG_REQUIRE(limit >= beams && limit <= vocab && vocab < (1 << 30), "beam_select: bad vocabulary");
    MG_REQUIRE(scratch != nullptr && ((uintptr_t)scratch & 15) == 0 && ((uintptr_t)logits & 3) == 0, "beam_select: scratch or alignment");
    const int rows = groups * in_beams, chunk = chunk_of(rows, limit), parts = parts_of(rows, limit);
    MG_REQUIRE(rows <= 65535, "beam_select: at most 65535 rows");
    u64* lists = (u64*)scratch;
    float* sums = (float*)(lists + (size_t)rows * parts * beams);
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e = mg_launch(beam_rows_kernel, dim3(parts, rows), dim3(ROW_THREADS), 0, s, true, logits, ended, lists, sums, vocab,
                              limit, beams, chunk);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "beam_select: %s", cudaGetErrorString(e));
    MG_CHECK_LAUNCH("beam_select");
    const ChoiceArgs a = {lists, sums, scores, ended, lengths, tokens, parents, scores_out, ranks, ended_out, lengths_out,
                          in_beams, beams, parts, end_token, penalty};
    int per_row = 1;
    while (2 * per_row * in_beams <= 32 && per_row < parts) per_row *= 2;
    // (it may start while the kernel in front of it, this operator's own, still runs)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(groups);
    cfg.blockDim = dim3(32 * per_row * in_beams);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, beam_choice_kernel, a);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "beam_select (choice): %s", cudaGetErrorString(e));
    MG_CHECK_LAUNCH("beam_select (choice)");
    return MG_OK;
}

// Rows whose parent is another row take over, from the parent: the block table's columns of full pages, the tokens of the
// part-filled page (into the row's own page of that column), and the state slot's contents.  parents, lengths, slots: [rows]
// ints on the device (lengths: tokens in the cache; slots may be null without states).  A parent has to be its own parent, as
// mg_beam_select leaves them: rows with another parent are left alone, as are rows whose parent is out of range or whose page
// is missing.
// paged: per group ten numbers (addresses of table, keys and values, layers, pages, kv heads, page tokens, bytes of a key, bytes
// of a value, table width); values 0: they live in the keys.  states: per tensor three (address, bytes of a slot, slots).
MG_API int mg_beam_reorder(const int* parents, const int* lengths, const int* slots, int rows, int n_paged, int n_states,
                           const long long* paged, const long long* states, void* stream) {
    if (rows == 0 || n_paged + n_states == 0) return MG_OK;
    MG_REQUIRE(rows > 0 && rows <= 65535 && n_paged >= 0 && n_paged <= MAX_PAGED && n_states >= 0 && n_states <= MAX_STATES,
               "beam_reorder: at most 65535 rows, %d groups of pages and %d states", MAX_PAGED, MAX_STATES);
    MG_REQUIRE((n_paged == 0 || lengths != nullptr) && (n_states == 0 || slots != nullptr), "beam_reorder: no lengths or no slots");
    ReorderArgs a = {};
    a.parents = parents; a.lengths = lengths; a.slots = slots; a.rows = rows; a.n_paged = n_paged; a.n_states = n_states;
    long long largest = 1;
    for (int g = 0; g < n_paged; ++g) {
        const long long* z = paged + 10 * g;
        for (int i = 3; i < 10; ++i) MG_REQUIRE(z[i] > 0 && z[i] < (1ll << 31), "beam_reorder: bad page sizes");
        Paged& p = a.paged[g];
        p.table = (int*)z[0]; p.k = (char*)z[1]; p.v = (char*)z[2];
        p.layers = (int)z[3]; p.num_pages = (int)z[4]; p.n_kv_head = (int)z[5]; p.page_tokens = (int)z[6];
        p.k_token = (int)z[7]; p.v_token = (int)z[8]; p.width = (int)z[9];
        p.k_layer = z[4] * z[5] * z[6] * z[7];
        p.v_layer = z[4] * z[5] * z[6] * z[8];
        p.unit = unit_of((uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.k_token | (uintptr_t)p.v_token);
        const long long bytes = z[3] * z[5] * z[6] * (z[7] + (p.v ? z[8] : 0));
        if (bytes > largest) largest = bytes;
    }
    for (int i = 0; i < n_states; ++i) {
        const long long* z = states + 3 * i;
        MG_REQUIRE(z[1] > 0 && z[2] > 0 && z[2] < (1ll << 31), "beam_reorder: bad state sizes");
        a.state[i] = {(char*)z[0], z[1], unit_of((uintptr_t)z[0] | (uintptr_t)z[1]), (int)z[2]};
        if (z[1] > largest) largest = z[1];
    }
    long long pieces = (largest + 32767) / 32768;
    if (pieces > 64) pieces = 64;
    const cudaError_t e = mg_launch(beam_reorder_kernel, dim3((unsigned)pieces, rows, n_paged + n_states), dim3(256), 0,
                                    (cudaStream_t)stream, true, a);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "beam_reorder: %s", cudaGetErrorString(e));
    MG_CHECK_LAUNCH("beam_reorder");
    return MG_OK;
}
