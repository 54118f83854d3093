// Attention of single query tokens over the paged cache where groups of tokens share their first keys: the beams of a
// search, the samples of one prompt.
//
// A row's result is the softmax average over the keys 0 .. its position, as in the other attention kernels; what differs is
// how often the keys are read.  Where every row reads all of its keys, a prompt of P tokens continued B times is read B
// times.  Here the keys are cut into ranges of two kinds: those of the P tokens that a group's rows share, read once for
// the (row, head) pairs of the group and key/value head that a CTA takes, and those behind them, read for their own row.
// (A CTA takes 256 pairs on tcgen05; on the warp-level tensor cores 32, at heads beyond 64 features 16, beyond 128 eight; in 32
// bits 16.  A group of more pairs has more CTAs, and each of them reads the shared keys.  32 rows of 2,000 shared tokens in a
// captured step, us, against every row reading its own: heads of 256, 8/2 (16 CTAs of eight pairs) 29 and 40, 8/8 (four) 39
// and 89; 8 x 8 rows of 1,021, 8/8 heads of 64 13 and 20, of 96 20 and 166, in 32 bits 55 and 68.)  A range leaves
// per (row, head) its unnormalised average acc, its maximum m (of the scores times log2 e) and its sum l, and a second
// kernel joins them:  M = max m_i,  out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
//
// How many ranges there are is the host's choice, from bounds on the lengths that it knows when it launches (a captured
// step has its grid for good); where the ranges lie is worked out on the device from the lengths as they are: a length is
// cut into as many ranges as there are, of at least a fixed number of keys, so bounds that are too low cost time only.  The
// same holds for the rows of a group.  A row that stands in front of the end of its group's shared tokens reads all its
// keys for itself, and so does one that belongs to no group.
//
// A range without keys (their pages are missing) leaves m = -inf and l = 0.  One whose keys all score -inf leaves m = -inf and
// l = 1: it counts for nothing beside others, and where there are no others the result is no number, as the softmax is.  Maxima
// pass over a score that is no number; l does not, and neither does the result.
#include <math.h>

#include "blackwell.cuh"
#include "tensor_map.cuh"
#include "warp_mma.cuh"

MG_GUARD_DECLARE(attention_shared)

namespace {

constexpr int BLOCK_KEYS = 64;         // keys of a block of the 32-bit kernel; ranges are cut at multiples of it (shared ones: see range_keys)

struct SharedArgs {
    const void* q;                     // rows whose first n_head * D columns are the queries
    long long q_stride;
    const void* k_pages;               // [page][kv head][token][D]
    const void* v_pages;
    const int* table;                  // [request][max_pages]
    const int* token_request;
    const int* positions;
    const int* groups;                 // [n_groups][3]: first row, rows, shared tokens
    void* out;                         // [n][n_head * D]
    float* part_out;                   // [row][head][slot][D]
    float* part_ml;                    // [row][head][slot][2]
    int* behind;                       // [row]: keys that its shared ranges hold (the ranges' kernel tells the joining one)
    int element;                       // bytes of a number of `out`
    int n_groups, n, n_head, n_kv_head, D, page_tokens, max_pages, num_pages, n_requests;
    int row_tiles;                     // CTAs that share the (row, head) pairs of a group
    int shared_slots, own_slots;       // ranges of the shared keys, and of a row's own
    int page_shift;                    // page_tokens as a power of two, -1: it is none
    int shared_least;                  // keys of a range of shared keys, at least, and what they are a multiple of
    int direct;                        // every row has one range alone: the results, not parts to be joined, are left
    int first_item;                    // item of the grid's first CTA: above 0 where another kernel takes the shared ranges
    float scale_log2e;
};

// Keys of one range when `keys` of them are cut into at most `slots`, each a multiple of `least` keys.
__device__ __forceinline__ int range_keys(int keys, int slots, int least) {
    const int even = (keys + slots - 1) / slots;
    return max(1, (even + least - 1) / least) * least;
}

constexpr int OWN_LEAST = 64;

// A group's shared tokens: a number that no row's block table reaches (or below zero) counts as none.
__device__ __forceinline__ int tokens_of(const SharedArgs& a, int group) {
    const int tokens = a.groups[3 * group + 2];
    return tokens < 0 || tokens > (long long)a.max_pages * a.page_tokens ? 0 : tokens;
}

// A row's position, at most the last that its block table reaches; below zero: padding.
__device__ __forceinline__ int position_of(const SharedArgs& a, int row) {
    const int p = a.positions[row];
    const long long last = (long long)a.max_pages * a.page_tokens - 1;
    return p > last ? (int)last : p;
}

// The shared tokens of the group that `row` belongs to (0: none); every warp finds them for itself.
__device__ __forceinline__ int group_tokens(const SharedArgs& a, int row) {
    const int lane = threadIdx.x & 31;
    int tokens = 0;
    for (int g0 = 0; g0 < a.n_groups; g0 += 32) {
        const int g = g0 + lane;
        bool mine = false;
        int shared = 0;
        if (g < a.n_groups) {
            const int first = a.groups[3 * g], rows = a.groups[3 * g + 1];
            shared = tokens_of(a, g);
            mine = first >= 0 && row >= first && row - first < rows;
        }
        const uint32_t found = __ballot_sync(0xffffffffu, mine);
        if (found) tokens = __shfl_sync(0xffffffffu, shared, __ffs(found) - 1);
    }
    return tokens;
}

// The request of the first of a group's rows that sees all its shared tokens, whose block table leads to them all (a row in
// front of their end, or one of padding, need not have their pages); -1: none does.  Whole warps call it.
__device__ __forceinline__ int sharing_request(const SharedArgs& a, int first_row, int rows, int tokens) {
    const int lane = threadIdx.x & 31;
    for (int r0 = 0; r0 < rows; r0 += 32) {
        const bool in = r0 + lane < rows;
        const int request = in ? a.token_request[first_row + r0 + lane] : 0;      // (asked for together with the position)
        const uint32_t found = __ballot_sync(0xffffffffu, in && position_of(a, first_row + r0 + lane) + 1 >= tokens);
        if (found) return __shfl_sync(0xffffffffu, request, __ffs(found) - 1);
    }
    return -1;
}

// What a CTA works on: (row, head) pairs of `rows` rows and the keys key0 .. key1 - 1 that their ranges `slot` hold.
struct Item {
    int first_row, rows, tile, tiles, key0, key1, slot, shared_keys;
    bool shared;
    const int* table;
};

// False if there is nothing to do.  Whole warps call it.
__device__ __forceinline__ bool item_of(const SharedArgs& a, int item, Item& it) {
    const int shared_items = a.n_groups * a.row_tiles * a.shared_slots;
    it.shared = item < shared_items;
    it.shared_keys = 0;
    it.tile = 0;
    it.tiles = it.rows = 1;
    int request;
    if (it.shared) {
        it.slot = item % a.shared_slots;
        item /= a.shared_slots;
        it.tile = item % a.row_tiles;
        it.tiles = a.row_tiles;
        const int g = item / a.row_tiles;
        it.first_row = a.groups[3 * g];
        it.rows = a.groups[3 * g + 1];
        it.shared_keys = tokens_of(a, g);
        if (it.first_row < 0 || it.rows <= 0 || it.first_row >= a.n) return false;
        it.rows = min(it.rows, a.n - it.first_row);
        request = sharing_request(a, it.first_row, it.rows, it.shared_keys);
        if (request < 0) return false;
        const int step = range_keys(it.shared_keys, a.shared_slots, a.shared_least);
        it.key0 = it.slot * step;
        it.key1 = min(it.shared_keys, it.key0 + step);
    } else {
        item -= shared_items;
        it.slot = item % a.own_slots;
        it.first_row = item / a.own_slots;
        const int p = position_of(a, it.first_row);
        request = a.token_request[it.first_row];
        int behind = group_tokens(a, it.first_row);
        if (behind > p + 1) behind = 0;
        if (a.direct) {
            if (p < 0) {                                  // padding of a fixed-size batch (else the joining kernel's work)
                const int size = a.n_head / a.n_kv_head * a.D * a.element;
                char* const out = (char*)a.out + ((size_t)it.first_row * a.n_kv_head + blockIdx.y) * size;
                for (int i = threadIdx.x; i < size; i += blockDim.x) out[i] = 0;
            }
        } else if (it.slot == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
            a.behind[it.first_row] = behind;
        }
        const int step = range_keys(p + 1 - behind, a.own_slots, OWN_LEAST);
        it.key0 = behind + it.slot * step;
        it.key1 = min(p + 1, it.key0 + step);
        it.slot += a.shared_slots;
    }
    if (!MG_GUARDED(attention_shared, MG_GUARD_REQUEST, request, a.n_requests)) request = 0;
    it.table = a.table + (size_t)request * a.max_pages;
    return it.key0 < it.key1;
}

// Row of the pool, seen as [page * kv head * token][D], of the key at a position; -1: it has no page (and is not there).
__device__ __forceinline__ int cache_row(const SharedArgs& a, const Item& it, int position, int kv_head) {
    if (position >= it.key1) return -1;
    const int pi = a.page_shift >= 0 ? position >> a.page_shift : position / a.page_tokens;
    int page = pi < a.max_pages ? it.table[pi] : -1;
    if (page >= 0 && !MG_GUARDED(attention_shared, MG_GUARD_PAGE, page, a.num_pages)) page = -1;
    if (page < 0 || page >= a.num_pages) return -1;
    return (page * a.n_kv_head + kv_head) * a.page_tokens + position - pi * a.page_tokens;
}

// The row of pair j of an item, or -1: pairs behind the last one, and rows that do not see all the shared keys.
__device__ __forceinline__ int pair_row(const SharedArgs& a, const Item& it, int j, int share) {
    if (j >= it.rows * share) return -1;
    const int row = it.first_row + j / share;
    return !it.shared || position_of(a, row) + 1 >= it.shared_keys ? row : -1;
}

// A row's result from its average, maximum and sum over all its keys (no key has a page: zeros).
__device__ __forceinline__ float result_of(float v, float top, float sum) {
    return sum == 0.f ? 0.f : top == -INFINITY ? NAN : v / sum;
}

// What a range leaves of feature d of a (row, head): the unnormalised average, with the maximum and the sum, or, where a row has one
// range alone, the result.
template <typename T>
__device__ __forceinline__ void leave(const SharedArgs& a, const Item& it, int row, int head, int d, float v, float top, float sum) {
    const size_t pair = (size_t)row * a.n_head + head;
    if (a.direct) {
        ((T*)a.out)[pair * a.D + d] = from_float<T>(result_of(v, top, sum));
        return;
    }
    const size_t at = pair * (a.shared_slots + a.own_slots) + it.slot;
    a.part_out[at * a.D + d] = v;
    if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(top, sum);
}

// ---- any head size, either type: 8 or 16 (row, head) pairs and 64 keys at a time, in 32-bit arithmetic -------------------
// The 32-bit mode's kernel, and that of bfloat16 heads whose size is no multiple of 8.  Keys and values of a block come to
// shared memory together, several loads a thread on their way (read one by one where they are used: 27 us for 10 rows of
// some 530 keys and 12 heads of 64, where this takes 14).  Scores: a thread a key and half of the pairs; average: a thread a
// feature and all pairs.
constexpr int SIMT_THREADS = 128;

__host__ __device__ constexpr int simt_lanes(int d) { return d > 64 ? 128 : d > 32 ? 64 : 32; }     // threads across the features

// Rows of a block into shared memory as 32-bit numbers; missing rows as zeros.  VEC: four features at a time.
template <typename T, bool VEC>
__device__ __forceinline__ void load_rows(const T* pages, const int* krow, float* to, int stride, int D) {
    constexpr int W = VEC ? 4 : 1;
    const int pieces = D / W, lanes = pieces > 16 ? 32 : pieces > 8 ? 16 : 8, at_once = SIMT_THREADS / lanes;
    const int r0 = threadIdx.x / lanes, c0 = threadIdx.x % lanes;
    for (int c = c0; c < pieces; c += lanes)
#pragma unroll 4
        for (int r = r0; r < BLOCK_KEYS; r += at_once) {
            const int row = krow[r];
            float v[W];
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = 0.f;
            if (row >= 0) {
                const T* from = pages + (size_t)row * D + c * W;
                if constexpr (VEC) {
                    const float4 x = *reinterpret_cast<const float4*>(from);
                    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
                } else {
                    v[0] = to_float(*from);
                }
            }
#pragma unroll
            for (int i = 0; i < W; ++i) to[r * stride + c * W + i] = v[i];
        }
}

template <typename T, int NQ, bool VEC>
__global__ void __launch_bounds__(SIMT_THREADS) attention_shared_simt_kernel(SharedArgs a) {
    extern __shared__ float4 smem4[];
    __shared__ int krow[BLOCK_KEYS], q_token[NQ], q_head[NQ];
    __shared__ float q_max[NQ], q_sum[NQ], q_corr[NQ];
    __shared__ int seen;                                 // whether the range has a key
    constexpr int HALF = NQ / 2;
    const int tid = threadIdx.x, D = a.D, kv_head = blockIdx.y, share = a.n_head / a.n_kv_head;
    float* q_s = reinterpret_cast<float*>(smem4);        // [D][NQ]
    float* p_s = q_s + D * NQ;                           // [64][NQ]
    float* v_s = p_s + BLOCK_KEYS * NQ;                  // [64][D]
    float* k_s = v_s + BLOCK_KEYS * D;                   // [64][D + 1]
    const int lanes = simt_lanes(D), dl = tid % lanes, ks = tid / lanes, key_parts = SIMT_THREADS / lanes;

    Item it;
    pdl_wait();
    pdl_trigger();
    if (!item_of(a, a.first_item + blockIdx.x, it)) return;
    for (int q0 = it.tile * NQ; q0 < it.rows * share; q0 += it.tiles * NQ) {
        __syncthreads();
        if (tid < NQ) {
            q_token[tid] = pair_row(a, it, q0 + tid, share);
            q_head[tid] = kv_head * share + (q0 + tid) % share;
            q_max[tid] = -INFINITY;
            q_sum[tid] = 0.f;
            seen = 0;
        }
        __syncthreads();
        for (int d = tid; d < D; d += SIMT_THREADS)
#pragma unroll
            for (int j = 0; j < NQ; ++j)
                q_s[d * NQ + j] = q_token[j] < 0 ? 0.f : to_float(((const T*)a.q)[q_token[j] * a.q_stride + (size_t)q_head[j] * D + d]) * a.scale_log2e;
        float acc[2][NQ];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NQ; ++j) acc[i][j] = 0.f;
        for (int b0 = it.key0; b0 < it.key1; b0 += BLOCK_KEYS) {
            __syncthreads();
            if (tid < BLOCK_KEYS) {
                krow[tid] = cache_row(a, it, b0 + tid, kv_head);
                if (krow[tid] >= 0) seen = 1;
            }
            __syncthreads();
            load_rows<T, VEC>((const T*)a.k_pages, krow, k_s, D + 1, D);
            load_rows<T, VEC>((const T*)a.v_pages, krow, v_s, D, D);
            __syncthreads();
            {
                const int key = tid & (BLOCK_KEYS - 1), j0 = (tid / BLOCK_KEYS) * HALF;
                float s[HALF];
#pragma unroll
                for (int j = 0; j < HALF; ++j) s[j] = 0.f;
#pragma unroll 4
                for (int d = 0; d < D; ++d) {
                    const float k = k_s[key * (D + 1) + d];
#pragma unroll
                    for (int j = 0; j < HALF; j += 4) {
                        const float4 q = *reinterpret_cast<const float4*>(q_s + d * NQ + j0 + j);
                        s[j] = fmaf(k, q.x, s[j]);
                        s[j + 1] = fmaf(k, q.y, s[j + 1]);
                        s[j + 2] = fmaf(k, q.z, s[j + 2]);
                        s[j + 3] = fmaf(k, q.w, s[j + 3]);
                    }
                }
#pragma unroll
                for (int j = 0; j < HALF; ++j) p_s[key * NQ + j0 + j] = krow[key] < 0 ? -INFINITY : s[j];
            }
            __syncthreads();
            if (tid < NQ * 8) {
                const int j = tid >> 3, part = tid & 7;              // eight neighbouring threads a query
                float x[BLOCK_KEYS / 8], m = -INFINITY;
#pragma unroll
                for (int k = 0; k < BLOCK_KEYS / 8; ++k) {
                    x[k] = p_s[(k * 8 + part) * NQ + j];
                    m = fmaxf(m, x[k]);
                }
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float before = q_max[j], top = fmaxf(before, m);
                float sum = 0.f;
#pragma unroll
                for (int k = 0; k < BLOCK_KEYS / 8; ++k) {
                    const float e = x[k] == -INFINITY ? 0.f : exp2f(x[k] - top);      // (no number stays none)
                    p_s[(k * 8 + part) * NQ + j] = e;
                    sum += e;
                }
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                __syncwarp();
                if (part == 0) {
                    const float corr = before == -INFINITY ? 0.f : exp2f(before - top);
                    q_corr[j] = corr;
                    q_max[j] = top;
                    q_sum[j] = fmaf(q_sum[j], corr, sum);
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < NQ; ++j) acc[i][j] *= q_corr[j];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int d = dl + i * SIMT_THREADS;
                if (d >= D) break;
#pragma unroll 4
                for (int k = ks; k < BLOCK_KEYS; k += key_parts) {
                    const float v = v_s[k * D + d];
#pragma unroll
                    for (int j = 0; j < NQ; j += 4) {
                        const float4 p = *reinterpret_cast<const float4*>(p_s + k * NQ + j);
                        acc[i][j] = fmaf(p.x, v, acc[i][j]);
                        acc[i][j + 1] = fmaf(p.y, v, acc[i][j + 1]);
                        acc[i][j + 2] = fmaf(p.z, v, acc[i][j + 2]);
                        acc[i][j + 3] = fmaf(p.w, v, acc[i][j + 3]);
                    }
                }
            }
        }
        // the threads that shared the keys of a feature meet (the key tile is free: scratch)
        if (key_parts > 1) {
            __syncthreads();
            if (ks > 0 && dl < D)
#pragma unroll
                for (int j = 0; j < NQ; ++j) k_s[((ks - 1) * NQ + j) * D + dl] = acc[0][j];
            __syncthreads();
            if (ks == 0 && dl < D)
                for (int other = 0; other < key_parts - 1; ++other)
#pragma unroll
                    for (int j = 0; j < NQ; ++j) acc[0][j] += k_s[(other * NQ + j) * D + dl];
        }
        if (ks == 0)
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
                if (q_token[j] < 0) continue;
                const float sum = q_max[j] == -INFINITY && q_sum[j] == 0.f && seen ? 1.f : q_sum[j];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (dl + i * SIMT_THREADS < D) leave<T>(a, it, q_token[j], q_head[j], dl + i * SIMT_THREADS, acc[i][j], q_max[j], sum);
            }
    }
}

// ---- bfloat16, heads of a multiple of 8 features: the warp-level tensor cores ------------------------------------------
// Keys are the rows of the products, pairs their columns (S = K q^T, 16 keys x 8 pairs; O = V^T P, 16 features x 8 pairs), so
// that a row's own keys, read for one pair or a few, waste little.  A CTA's four warps take 16 keys in turn; each copies its
// own rows from their pages (cp.async, a ring of stages), and keeps maximum, sum and average of its own, so the loop has no
// barrier.  The maximum is a reference that moves only when a score is more than 2^REF_SLACK above it: then everything so
// far is rescaled.  P goes into the product rounded to bfloat16 (2^-8 of a weight at most) for the heads whose weights the kernels of
// unshared keys round so (16, 32, 64, 128 and 256 features); for the others, where those hold more, as two bfloat16 numbers (FULL:
// 2^-16 of a weight).  The sums are of the 32-bit weights.
constexpr float REF_SLACK = 8.f;

// The 32-bit values of a pair's numbers.
__device__ __forceinline__ float bf16_low(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float bf16_high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

constexpr int MMA_THREADS = 128, MMA_WARPS = MMA_THREADS / 32, UNIT = 16;       // keys a warp takes at a time

// Sizes by padded head: DP features (32, 64, 128 or 256), of which D are there and the others zero; and the CTAs that an SM is to
// hold.  A CTA of few keys is mostly its chain of trips to memory (which range, its group, the pages, the keys), so many small
// rings an SM hide more than deep ones: heads of 64 at six CTAs of two stages instead of four of three 13.7 -> 11.6 us for 64 rows
// of 1,021 tokens.  Heads of 128 take one stage at six CTAs (MANY) or two at three: see cut().
template <int DP, int NT, bool MANY>
struct MmaSizes {
    static constexpr int STAGES = DP == 32 ? 4 : DP == 64 ? (NT == 1 ? 2 : 3) : MANY ? 1 : 2;
    static constexpr int CTAS = DP == 32 ? (NT == 1 ? 8 : NT == 2 ? 5 : 4) : DP == 64 ? (NT == 1 ? 6 : NT == 2 ? 4 : 3) : MANY ? 6 : DP == 128 && NT == 1 ? 3 : 2;
    static constexpr int TILE = UNIT * DP * 2;                          // bytes of 16 keys or values
    static constexpr size_t SMEM = (size_t)MMA_WARPS * STAGES * 2 * TILE;
};

template <int DP, int NT, bool MANY, bool FULL>      // NT: tiles of 8 pairs that a CTA takes at once
__global__ void __launch_bounds__(MMA_THREADS, MmaSizes<DP, NT, MANY>::CTAS) attention_shared_mma_kernel(SharedArgs a) {
    using Z = MmaSizes<DP, NT, MANY>;
    constexpr int STAGES = Z::STAGES, CPR = DP / 8, ROWB = 2 * DP;
    constexpr int RPL = CPR >= 8 ? 1 : 8 / CPR, SWZ = CPR >= 8 ? 8 : CPR;     // piece c of row r lies at piece c ^ ((r / RPL) % SWZ)
    constexpr int PSTRIDE = DP + 2;                                     // floats of a warp's partial: O, maximum, sum
    static_assert((size_t)MMA_WARPS * NT * 8 * PSTRIDE * 4 <= Z::SMEM, "the warps' results meet where the tiles were");
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint32_t valid[MMA_WARPS][STAGES];
    __shared__ int pair_token[NT * 8], pair_head[NT * 8];
    __shared__ float weight[MMA_WARPS][NT * 8], pair_top[NT * 8], pair_sum[NT * 8];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int kv_head = blockIdx.y, share = a.n_head / a.n_kv_head, D = a.D, pieces = D / 8;
    const bf16* const k_pages = (const bf16*)a.k_pages;
    const bf16* const v_pages = (const bf16*)a.v_pages;
    Item it;
    // Behind the kernel of the shared ranges this one starts while that still runs: what both read was there before that one
    // let it start.  It ends behind that one (the joining kernel waits for this kernel alone).
    if (a.first_item == 0) pdl_wait();
    pdl_trigger();
    if (!item_of(a, a.first_item + blockIdx.x, it)) {
        if (a.first_item > 0) pdl_wait();
        return;
    }
    uint8_t* const mine = ring + (size_t)warp * STAGES * 2 * Z::TILE;
    const uint32_t mine_u = (uint32_t)__cvta_generic_to_shared(mine);
    const uint4 zero4 = make_uint4(0u, 0u, 0u, 0u);
    const int units = (it.key1 - it.key0 + UNIT - 1) / UNIT, my_units = units > warp ? (units - warp + MMA_WARPS - 1) / MMA_WARPS : 0;

    for (int q0 = it.tile * NT * 8; q0 < it.rows * share; q0 += it.tiles * NT * 8) {
        const int nts = min(NT, (it.rows * share - q0 + 7) / 8);       // tiles of pairs that there are
        if (pieces < CPR) {                                             // features that are not there: zeros in every stage
            for (int i = lane; i < STAGES * 2 * UNIT * (CPR - pieces); i += 32) {
                const int r = i / (CPR - pieces), c = pieces + i % (CPR - pieces);
                *reinterpret_cast<uint4*>(mine + r * ROWB + ((c ^ (((r % UNIT) / RPL) % SWZ)) * 16)) = zero4;
            }
        }
        // the first units' rows of the pool, then the copies; the rows of the unit after the last one asked for are on their way
        auto row_of = [&](int n) {                                      // lane i: row of key i of this warp's n-th unit
            return n < my_units ? cache_row(a, it, it.key0 + (warp + n * MMA_WARPS) * UNIT + (lane & 15), kv_head) : -1;
        };
        auto load = [&](int n, int row) {
            if (n < my_units) {
                const uint32_t there = __ballot_sync(0xffffffffu, row >= 0) & 0xffffu;
                if (lane == 0) valid[warp][n % STAGES] = there;
                const uint32_t at = (uint32_t)(n % STAGES) * 2 * Z::TILE;
#pragma unroll
                for (int i0 = 0; i0 < UNIT * CPR; i0 += 32) {
                    const int i = i0 + lane, r = i / CPR, c = i % CPR;
                    const int from = __shfl_sync(0xffffffffu, row, r);
                    const uint32_t off = at + r * ROWB + ((c ^ ((r / RPL) % SWZ)) * 16);
                    if (c < pieces) {
                        if (from >= 0) {
                            cp_async16(mine_u + off, k_pages + (size_t)from * D + c * 8);
                            cp_async16(mine_u + off + Z::TILE, v_pages + (size_t)from * D + c * 8);
                        } else {                                        // keeps 0 * garbage out of the product
                            *reinterpret_cast<uint4*>(mine + off) = zero4;
                            *reinterpret_cast<uint4*>(mine + off + Z::TILE) = zero4;
                        }
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int row = row_of(0);
#pragma unroll
        for (int n = 0; n < STAGES; ++n) {
            const int next = row_of(n + 1);
            load(n, row);
            row = next;
        }
        // the pairs' queries as the B operand: pair nt * 8 + g in column g
        uint32_t qb[NT][DP / 16][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int j = q0 + nt * 8 + g, token = nt < nts ? pair_row(a, it, j, share) : -1;
            const bf16* const q = (const bf16*)a.q + (token < 0 ? 0 : token * a.q_stride + (size_t)(kv_head * share + j % share) * D);
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int d = ks * 16 + h * 8 + 2 * t;
                    qb[nt][ks][h] = token >= 0 && d < D ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
                }
        }
        float o[NT][DP / 16][4], ref[NT][2], sum[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            ref[nt][0] = ref[nt][1] = -INFINITY;
            sum[nt][0] = sum[nt][1] = 0.f;
#pragma unroll
            for (int dm = 0; dm < DP / 16; ++dm)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[nt][dm][i] = 0.f;
        }
        // ldmatrix addresses: K as the A operand (matrix j = lane / 8: keys (j % 2) * 8 .., piece j / 2), V transposed (keys
        // (j / 2) * 8 .., piece j % 2)
        const int krow = (lane & 7) + (((lane >> 3) & 1) << 3), kpiece = lane >> 4;
        const int vrow = (lane & 7) + (((lane >> 4) & 1) << 3), vpiece = (lane >> 3) & 1;
        uint32_t seen = 0;                                              // whether this warp had a key
        for (int n = 0; n < my_units; ++n) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();                                               // this unit has landed
            const int next = row_of(n + STAGES + 1);
            const uint32_t k_at = mine_u + (uint32_t)(n % STAGES) * 2 * Z::TILE, v_at = k_at + Z::TILE;
            const uint32_t there = valid[warp][n % STAGES];
            seen |= there;
            float s[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
            for (int ks = 0; ks < DP / 16; ++ks) {
                uint32_t f[4];
                ldmatrix_x4(f, k_at + krow * ROWB + (((ks * 2 + kpiece) ^ ((krow / RPL) % SWZ)) * 16));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (nt < nts) mma_bf16(s[nt], f, qb[nt][ks][0], qb[nt][ks][1]);
            }
            // a lane holds pairs 2t, 2t+1 (numbers 0, 1 and 2, 3) of keys g and g + 8
            bool above = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[nt][i] = (there >> (g + ((i >> 1) << 3))) & 1u ? s[nt][i] * a.scale_log2e : -INFINITY;
                    above = above || (nt < nts && !(s[nt][i] <= ref[nt][i & 1] + REF_SLACK));
                }
            if (__any_sync(0xffffffffu, above)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float top = fmaxf(ref[nt][i], fmaxf(s[nt][i], s[nt][i + 2]));
#pragma unroll
                        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                        const float corr = ref[nt][i] == -INFINITY ? 0.f : exp2f(ref[nt][i] - top);
                        ref[nt][i] = top;
                        sum[nt][i] *= corr;
#pragma unroll
                        for (int dm = 0; dm < DP / 16; ++dm) {
                            o[nt][dm][i] *= corr;
                            o[nt][dm][i + 2] *= corr;
                        }
                    }
            }
            uint32_t pb[NT][2], rest[NT][2];                           // the weights, and what their rounding leaves
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    e[i] = exp2_approx(s[nt][i] - (ref[nt][i & 1] == -INFINITY ? 0.f : ref[nt][i & 1]));
                    sum[nt][i & 1] += e[i];
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t p = pack_bf16(e[2 * h], e[2 * h + 1]);
                    pb[nt][h] = movmatrix_trans(p);
                    if constexpr (FULL) rest[nt][h] = movmatrix_trans(pack_bf16(e[2 * h] - bf16_low(p), e[2 * h + 1] - bf16_high(p)));
                }
            }
#pragma unroll
            for (int dm = 0; dm < DP / 16; ++dm) {
                uint32_t f[4];
                ldmatrix_x4_trans(f, v_at + vrow * ROWB + (((dm * 2 + vpiece) ^ ((vrow / RPL) % SWZ)) * 16));
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                    if (nt < nts) {
                        mma_bf16(o[nt][dm], f, pb[nt][0], pb[nt][1]);
                        if constexpr (FULL) mma_bf16(o[nt][dm], f, rest[nt][0], rest[nt][1]);
                    }
            }
            __syncwarp();                                               // the unit is used up
            load(n + STAGES, row);
            row = next;
        }
        // the warps' results meet in shared memory
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();
        float* const part = reinterpret_cast<float*>(ring);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) sum[nt][i] += __shfl_xor_sync(0xffffffffu, sum[nt][i], x);
                float* const dst = part + (warp * NT * 8 + nt * 8 + 2 * t + i) * PSTRIDE;
#pragma unroll
                for (int dm = 0; dm < DP / 16; ++dm) {
                    dst[dm * 16 + g] = o[nt][dm][i];
                    dst[dm * 16 + g + 8] = o[nt][dm][i + 2];
                }
                if (g == 0) {
                    dst[DP] = ref[nt][i];
                    dst[DP + 1] = ref[nt][i] == -INFINITY && sum[nt][i] == 0.f && seen ? 1.f : sum[nt][i];
                }
            }
        __syncthreads();
        // a pair's row and head, and what each warp's numbers count for
        if (tid < NT * 8) {
            pair_token[tid] = tid < nts * 8 ? pair_row(a, it, q0 + tid, share) : -1;
            pair_head[tid] = kv_head * share + (q0 + tid) % share;
            float top = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < MMA_WARPS; ++w) top = fmaxf(top, part[(w * NT * 8 + tid) * PSTRIDE + DP]);
#pragma unroll
            for (int w = 0; w < MMA_WARPS; ++w) {                       // warps in order
                const float ref_w = part[(w * NT * 8 + tid) * PSTRIDE + DP];
                const float f = ref_w != -INFINITY ? exp2f(ref_w - top) : top == -INFINITY ? 1.f : 0.f;
                weight[w][tid] = f;
                l = fmaf(f, part[(w * NT * 8 + tid) * PSTRIDE + DP + 1], l);
            }
            pair_top[tid] = top;
            pair_sum[tid] = l;
        }
        __syncthreads();
        for (int j = warp; j < nts * 8; j += MMA_WARPS) {
            const int token = pair_token[j];
            if (token < 0) continue;
            for (int d = lane; d < D; d += 32) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < MMA_WARPS; ++w) v = fmaf(weight[w][j], part[(w * NT * 8 + j) * PSTRIDE + d], v);
                leave<bf16>(a, it, token, pair_head[j], d, v, pair_top[j], pair_sum[j]);
            }
        }
        __syncthreads();                                                // (the tiles are loaded again for the next pairs)
    }
    if (a.first_item > 0) pdl_wait();
}

// ---- bfloat16, heads of 64 or 128, many pairs: the 5th-generation tensor cores --------------------------------------------
// A CTA takes two tiles of 128 pairs and walks over the keys of its range in blocks of 64, which both tiles multiply with:
//
//   load warp       TMA tiles of keys and values from the pages (one copy per page, tensor and 64 features, 128-byte swizzle)
//                   into a ring of stages
//   issue warps     one a tile: S = Q K^T (128 x 64, one of two TMEM buffers), and O += P V (128 x head, TMEM) with P read from
//                   TMEM, where it lies in S's place.  The scores of a block are computed while the softmax is at the one before.
//   softmax warps   eight a tile, two threads a pair, each with half of its row of S: into registers, 2^(s - ref) as bfloat16
//                   back, the 32-bit sum kept.  `ref` is the first block's maximum and moves only when a block's sum is above 2^60
//                   (or no number): O is then rescaled in TMEM, and the block done again.  (O / sum does not depend on ref while
//                   the numbers are in range.)
//
// What bounds it: at heads of 128 a block is 2 x 128 x 64 x 128 multiply-adds a tile, 512 cycles of the tensor core (more for S,
// whose operands are both read from shared memory), and 8,192 exponentials, 512 cycles of the special-function units.  All waits
// for the tensor core and for copies are bounded: when one runs out, `status` gets a code, the CTA writes nothing more, frees
// its TMEM and returns.  (Blocks of 128 keys with one buffer a tile, a tile's softmax and products one after the other: 95 us
// where this takes 81 for 256 rows of 16,384 keys and 32/8 heads of 128.)
constexpr int TC_KEYS = 64, TC_PAIRS = 128, TC_TILES = 2;
constexpr int TC_SOFTMAX_WARPS = 8 * TC_TILES, TC_ISSUE = TC_SOFTMAX_WARPS, TC_LOAD = TC_ISSUE + TC_TILES, TC_THREADS = 32 * (TC_LOAD + 1);
constexpr uint32_t TC_COLS = 512, TC_O_COL = TC_TILES * 2 * TC_KEYS;      // S of both tiles and buffers, then O of both
constexpr float TC_LIMIT = 1.152921504606846976e18f;                     // 2^60: a block's sum above it moves the reference

template <int D>
struct TcSizes {
    static constexpr int ATOMS = D / 64, Q_ATOM = TC_PAIRS * 128, ATOM = TC_KEYS * 128;      // 64 features of a tile's rows, in bytes
    static constexpr int Q_TILE = ATOMS * Q_ATOM, TILE = ATOMS * ATOM, STAGES = 4;
    static constexpr size_t SMEM = 1024 + (size_t)TC_TILES * Q_TILE + (size_t)2 * STAGES * TILE;
};

struct __align__(8) TcSync {
    uint64_t kv_full[4], kv_free[4], s_full[TC_TILES][2], p_ready[TC_TILES][2], pv_done[TC_TILES], q_ready[TC_TILES], round_done[TC_TILES];
    float meet[TC_TILES][2][TC_PAIRS];      // what the two threads of a pair tell each other
    uint32_t tmem, failed;
};

// 32 lanes x 16 columns of 32-bit numbers.
__device__ __forceinline__ void tmem_load_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
// ... and 8.
__device__ __forceinline__ void tmem_load_8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_store_8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};"
                 ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr) : "memory");
}

// D[tmem] (+)= A[tmem] B, A's bfloat16 numbers two a column.
__device__ __forceinline__ void umma_bf16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
        ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
        : "memory");
}

template <int D>
__global__ void __launch_bounds__(TC_THREADS, 1)
attention_shared_tc_kernel(SharedArgs a, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                           int box_rows, int* __restrict__ status) {
    using Z = TcSizes<D>;
    constexpr int STAGES = Z::STAGES, ATOMS = Z::ATOMS;
    extern __shared__ uint8_t smem_raw[];
    __shared__ TcSync sync;
    uint8_t* const smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* const q_tiles = smem;
    uint8_t* const k_tiles = q_tiles + TC_TILES * Z::Q_TILE;
    uint8_t* const v_tiles = k_tiles + STAGES * Z::TILE;
    // (told by one lane to all: the compiler then knows that the warp agrees, which the tensor core's operands have to)
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int kv_head = blockIdx.y, share = a.n_head / a.n_kv_head;
    Item it;
    pdl_wait();                                                         // (before the next kernel may start: see there)
    pdl_trigger();
    if (!item_of(a, blockIdx.x, it)) return;                   // (shared ranges only: the grid has no others)
    const int n_blocks = (it.key1 - it.key0 + TC_KEYS - 1) / TC_KEYS, pairs = it.rows * share;
    const int boxes = TC_KEYS / box_rows, box_shift = __ffs(box_rows) - 1;       // (a power of two)
    auto page_at = [&](int column) {                                    // -1: none (its keys are not there)
        int page = column < a.max_pages ? it.table[column] : -1;
        if (page >= 0 && !MG_GUARDED(attention_shared, MG_GUARD_PAGE, page, a.num_pages)) page = -1;
        return page < a.num_pages ? page : -1;
    };

    if (tid == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&sync.kv_full[s]), 1);
            mbar_init(smem_u32(&sync.kv_free[s]), TC_TILES);
        }
        for (int i = 0; i < TC_TILES; ++i) {
            mbar_init(smem_u32(&sync.pv_done[i]), 1);
            for (int b = 0; b < 2; ++b) {
                mbar_init(smem_u32(&sync.s_full[i][b]), 1);
                mbar_init(smem_u32(&sync.p_ready[i][b]), 256);
            }
            mbar_init(smem_u32(&sync.q_ready[i]), 256);
            mbar_init(smem_u32(&sync.round_done[i]), 1);
        }
        sync.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TC_ISSUE) tmem_alloc(smem_u32(&sync.tmem), TC_COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sync.tmem, 0);
    const int round_pairs = TC_TILES * TC_PAIRS, first_pair = it.tile * round_pairs, stride = it.tiles * round_pairs;
    // (one round of pairs, unless the bound on a group's rows was too low; the barriers' phases go on counting)

    if (warp < TC_SOFTMAX_WARPS) {
        // warp: tile i, half h of the keys (and of the features), rows 32 * (warp % 4) .. of the tile
        constexpr int HALF = TC_KEYS / 2, DH = D / 2;
        const int i = warp / 8, h = (warp / 4) & 1, mine = tid & 127, pair_bar = 1 + i * 4 + (warp & 3);
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const uint32_t o_at = lanes + TC_O_COL + i * D + h * DH;
        // Whether any of the `threads` threads that meet at a barrier says so.  (All of them come to it, whatever they waited for in
        // vain: a wait that ran out is told here, and all leave together.)
        auto any_of = [&](int barrier, int threads, bool v) {
            uint32_t any;
            asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                         : "=r"(any) : "r"((uint32_t)v), "r"(barrier), "r"(threads) : "memory");
            return any != 0u;
        };
        // the other half's number (the two warps of 32 pairs meet)
        auto other_half = [&](float v) {
            sync.meet[i][h][mine] = v;
            asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
            const float w = sync.meet[i][h ^ 1][mine];
            asm volatile("bar.sync %0, 64;" ::"r"(pair_bar) : "memory");
            return w;
        };
        int n = 0, code = 0;                                            // blocks so far
        bool holes = false, looked = false, seen = false;               // whether a page of the range is missing, one is there
        for (int q0 = first_pair, round = 0; q0 < pairs && code == 0; q0 += stride, ++round) {
            const int j0 = q0 + i * TC_PAIRS;
            if (j0 >= pairs) continue;                                  // no pairs for this tile
            // queries: a pair a row of the tile, swizzled (pairs that are not there: zeros); a warp its 32 rows, all of a row's
            // pieces by neighbouring lanes
            const int row = pair_row(a, it, j0 + mine, share), head = kv_head * share + (j0 + mine) % share;
            const long long q_at = row < 0 ? -1 : row * a.q_stride + (long long)head * D;
#pragma unroll
            for (int e = h * (D / 16); e < (h + 1) * (D / 16); ++e) {
                constexpr int ROWS = 256 / D;                           // rows at once: 32 lanes of 8 features
                const int r = e * ROWS + lane / (D / 8), c = lane % (D / 8);
                const long long from = __shfl_sync(0xffffffffu, q_at, r);
                uint4 v = make_uint4(0u, 0u, 0u, 0u);
                if (from >= 0) v = *reinterpret_cast<const uint4*>((const bf16*)a.q + from + c * 8);
                *reinterpret_cast<uint4*>(q_tiles + i * Z::Q_TILE + (c / 8) * Z::Q_ATOM + ((warp & 3) * 32 + r) * 128 + (((c % 8) ^ (r & 7)) * 16)) = v;
            }
            async_proxy_fence();
            tc_fence_before();
            mbar_arrive(smem_u32(&sync.q_ready[i]));
            if (!looked) {                                              // (while the first keys are on their way)
                for (int c = it.key0 / a.page_tokens + lane; c <= (it.key1 - 1) / a.page_tokens; c += 32) {
                    const bool hole = page_at(c) < 0;
                    holes = holes || hole;
                    seen = seen || !hole;
                }
                holes = __any_sync(0xffffffffu, holes);
                seen = __any_sync(0xffffffffu, seen);
                looked = true;
            }
            float ref = -INFINITY, total = 0.f;
            for (int b = 0; b < n_blocks; ++b, ++n) {
                const int last = it.key1 - it.key0 - b * TC_KEYS;       // keys of this block
                const uint32_t buffer = lanes + (i * 2 + (n & 1)) * TC_KEYS, s_at = buffer + h * HALF;      // (P of a half: in front)
                if (code == 0 && !warp_wait(smem_u32(&sync.s_full[i][n & 1]), (n >> 1) & 1)) code = 64;
                tc_fence_after();
                uint32_t s[HALF];
#pragma unroll
                for (int c = 0; c < HALF / 32; ++c) tmem_load_32(s_at + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&s[c * 32]));
                tmem_wait_ld();
                if (last < TC_KEYS || holes) {
                    // keys behind the range's end, and those whose page is missing
                    const int position = it.key0 + b * TC_KEYS + lane * box_rows;
                    const uint32_t there = __ballot_sync(0xffffffffu, lane < boxes && position < it.key1 && page_at(position / a.page_tokens) >= 0);
#pragma unroll
                    for (int c = 0; c < HALF; ++c)
                        if (h * HALF + c >= last || !((there >> ((h * HALF + c) >> box_shift)) & 1u)) s[c] = 0xff800000u;
                }
                bool move = ref == -INFINITY;
                float sum = 0.f;
#pragma unroll 1
                for (int pass = 0; pass < 3; ++pass) {
                    if (pass > 0 || __any_sync(0xffffffffu, move)) {        // (the two threads of a pair agree on ref)
                        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, corr = 1.f;
#pragma unroll
                        for (int c = 0; c < HALF; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(s[c]));
                        float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.scale_log2e;
                        top = fmaxf(top, other_half(top));
                        move = other_half(move ? 1.f : 0.f) != 0.f || move;
                        if (move) {
                            corr = ref == -INFINITY ? 1.f : exp2f(ref - top);      // (nothing was summed before the first)
                            ref = top;
                        }
                        total *= corr;
                        if (b > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
                            // once the block before is in the average (that the one before it is, these scores have shown)
                            if (!warp_wait(smem_u32(&sync.pv_done[i]), (n - 1) & 1)) code = 68;
                            tc_fence_after();
#pragma unroll
                            for (int c = 0; c < DH / 8; ++c) {
                                uint32_t r[8];
                                tmem_load_8(o_at + c * 8, r);
                                tmem_wait_ld();
#pragma unroll
                                for (int k = 0; k < 8; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * corr);
                                tmem_store_8(o_at + c * 8, r);
                            }
                        }
                    }
                    // P in the scores' place, and the row's sum
                    const float shift = ref == -INFINITY ? 0.f : ref;
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int w = 0; w < HALF / 16; ++w) {
                        uint32_t p[8];
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const float e0 = exp2_approx(fmaf(__uint_as_float(s[w * 16 + 2 * c]), a.scale_log2e, -shift));
                            const float e1 = exp2_approx(fmaf(__uint_as_float(s[w * 16 + 2 * c + 1]), a.scale_log2e, -shift));
                            part[c & 3] += e0 + e1;
                            p[c] = pack_bf16(e0, e1);
                        }
                        tmem_store_8(s_at + w * 8, p);
                    }
                    sum = (part[0] + part[1]) + (part[2] + part[3]);
                    move = !(sum <= TC_LIMIT);
                    if (!any_of(pair_bar, 64, move || code != 0)) break;
                    if (other_half(code != 0 ? 1.f : 0.f) != 0.f && code == 0) code = 71;       // the other warp waited in vain
                }
                if (code != 0) break;                                   // (the same in both warps)
                total += sum;
                // value rows behind the range's last key hold whatever is in the page: 0 times that has to be 0 (both tiles write
                // the same zeros: neither waits for the other)
                if (last < TC_KEYS && h == 0) {
                    const int stage = n % STAGES;
                    if (!warp_wait(smem_u32(&sync.kv_full[stage]), (n / STAGES) & 1)) code = 65;
                    if (mine >= last && mine < TC_KEYS)
#pragma unroll
                        for (int atom = 0; atom < ATOMS; ++atom)
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                *reinterpret_cast<uint4*>(v_tiles + stage * Z::TILE + atom * Z::ATOM + mine * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
                    async_proxy_fence();
                }
                tmem_wait_st();
                tc_fence_before();
                mbar_arrive(smem_u32(&sync.p_ready[i][n & 1]));
            }
            // (a barrier of its own: pv_done may be two phases behind here, and their parities are alike)
            if (code == 0 && !warp_wait(smem_u32(&sync.round_done[i]), round & 1)) code = 66;
            tc_fence_after();
            // the averages: 16 features at a time by way of the tile's queries' place, so that neighbouring lanes write
            // neighbouring numbers
            const bool write = row >= 0 && code == 0 && *(volatile uint32_t*)&sync.failed == 0;
            const long long at = write ? ((long long)row * a.n_head + head) * (a.shared_slots + a.own_slots) + it.slot : -1;
            float4* const scratch = reinterpret_cast<float4*>(q_tiles + i * Z::Q_TILE + (warp & 7) * 2048);
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
                uint32_t r[16];
                tmem_load_16(o_at + c * 16, r);
                tmem_wait_ld();
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    scratch[lane * 4 + (k ^ ((lane >> 1) & 3))] = make_float4(__uint_as_float(r[4 * k]), __uint_as_float(r[4 * k + 1]),
                                                                              __uint_as_float(r[4 * k + 2]), __uint_as_float(r[4 * k + 3]));
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int from = k * 8 + lane / 4, piece = lane & 3;
                    const long long to = __shfl_sync(0xffffffffu, at, from);
                    if (to >= 0)
                        *reinterpret_cast<float4*>(a.part_out + to * D + h * DH + c * 16 + piece * 4) = scratch[from * 4 + (piece ^ ((from >> 1) & 3))];
                }
            }
            total += other_half(total);
            if (ref == -INFINITY && total == 0.f && seen) total = 1.f;
            if (write && h == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(ref, total);
            // (the queries' place is scratch no more)
            if (any_of(9 + i, 256, code != 0) && code == 0) code = 69;
        }
        if (code) {
            atomicExch(status, code);
            *(volatile uint32_t*)&sync.failed = 1;
        }
    } else {
        int code = 0;
        if (warp == TC_LOAD) {
            int n = 0;
            for (int q0 = first_pair; q0 < pairs && code == 0; q0 += stride) {
                // box `lane` of the blocks; its page is looked up a block ahead (pages smaller than a block: a box each; larger
                // ones begin at a block)
                int position = it.key0 + lane * box_rows, column = position / a.page_tokens, offset = position - column * a.page_tokens;
                auto look = [&]() { return lane < boxes && position < it.key1 && column < a.max_pages ? it.table[column] : -1; };
                int page = look();
                for (int b = 0; b < n_blocks && code == 0; ++b, ++n) {
                    const int stage = n % STAGES;
                    if (page >= a.num_pages) page = -1;
                    if (page >= 0 && !MG_GUARDED(attention_shared, MG_GUARD_PAGE, page, a.num_pages)) page = -1;
                    // (no page: rows in front of the pool, which the copy fills with zeros)
                    const int y = page < 0 ? -box_rows : (page * a.n_kv_head + kv_head) * a.page_tokens + offset;
                    position += TC_KEYS;
                    if (a.page_tokens < TC_KEYS) column += boxes;
                    else if ((offset += TC_KEYS) >= a.page_tokens) { offset = 0; ++column; }
                    page = look();
                    if (n >= STAGES && !warp_wait(smem_u32(&sync.kv_free[stage]), (n / STAGES - 1) & 1)) { code = 60; break; }
                    const uint32_t full = smem_u32(&sync.kv_full[stage]);
                    if (lane == 0) mbar_expect_tx(full, 2 * Z::TILE);
                    __syncwarp();
                    if (lane < boxes)
#pragma unroll
                        for (int atom = 0; atom < ATOMS; ++atom) {
                            const uint32_t off = stage * Z::TILE + atom * Z::ATOM + lane * box_rows * 128;
                            tma_load_2d(smem_u32(k_tiles) + off, &map_k, full, atom * 64, y);
                            tma_load_2d(smem_u32(v_tiles) + off, &map_v, full, atom * 64, y);
                        }
                    __syncwarp();
                }
            }
        } else if (elect_one()) {
            // One thread a tile issues its products and waits for its own softmax and products alone, so that the other tile's
            // fill the time.
            const int i = warp - TC_ISSUE;
            int n = 0;
            for (int q0 = first_pair, round = 0; q0 < pairs && code == 0; q0 += stride, ++round) {
                auto scores = [&](int m) {                              // S of block m = Q K^T, once its keys and values are there
                    const int stage = m % STAGES;
                    if (!mbar_wait(smem_u32(&sync.kv_full[stage]), (m / STAGES) & 1)) return false;
                    tc_fence_after();
                    constexpr uint32_t idesc = instr_desc_bf16(TC_PAIRS, TC_KEYS, false);
                    const uint64_t dq = smem_desc_sw128(smem_u32(q_tiles + i * Z::Q_TILE)), dk = smem_desc_sw128(smem_u32(k_tiles + stage * Z::TILE));
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_bf16(tmem + (i * 2 + (m & 1)) * TC_KEYS, dq + (uint64_t)((k / 4 * Z::Q_ATOM + k % 4 * 32) >> 4),
                                  dk + (uint64_t)((k / 4 * Z::ATOM + k % 4 * 32) >> 4), idesc, k ? 1u : 0u);
                    umma_commit(smem_u32(&sync.s_full[i][m & 1]));
                    return true;
                };
                if (q0 + i * TC_PAIRS >= pairs) {                       // no pairs for this tile: it gives the blocks back unread
                    for (int b = 0; b < n_blocks && code == 0; ++b, ++n) {
                        if (!mbar_wait(smem_u32(&sync.kv_full[n % STAGES]), (n / STAGES) & 1)) code = 61;
                        else mbar_arrive(smem_u32(&sync.kv_free[n % STAGES]));
                    }
                    continue;
                }
                if (!mbar_wait(smem_u32(&sync.q_ready[i]), round & 1)) { code = 67; break; }
                if (!scores(n) || (n_blocks > 1 && !scores(n + 1))) code = 61;
                for (int b = 0; b < n_blocks && code == 0; ++b, ++n) {
                    const int stage = n % STAGES;
                    if (!mbar_wait(smem_u32(&sync.p_ready[i][n & 1]), (n >> 1) & 1)) { code = 62; break; }
                    tc_fence_after();
                    constexpr uint32_t idesc = instr_desc_bf16(TC_PAIRS, D, true);
                    // (values: atoms of 64 features, the second an atom's bytes behind the first)
                    const uint64_t dv = smem_desc_sw128(smem_u32(v_tiles + stage * Z::TILE)) + ((uint64_t)((Z::ATOM >> 4) - 1) << 16);
#pragma unroll
                    for (int k = 0; k < TC_KEYS / 16; ++k)
                        umma_bf16_ts(tmem + TC_O_COL + i * D, tmem + (i * 2 + (n & 1)) * TC_KEYS + (k / 2) * (TC_KEYS / 2) + (k % 2) * 8,
                                     dv + (uint64_t)(k * (16 * 128) >> 4), idesc, (b | k) ? 1u : 0u);
                    umma_commit(smem_u32(&sync.pv_done[i]));
                    umma_commit(smem_u32(&sync.kv_free[stage]));
                    if (b == n_blocks - 1) umma_commit(smem_u32(&sync.round_done[i]));
                    // the scores of the block after the next, in the place of the P that has just gone into the average (only the wait
                    // orders the two)
                    if (b + 2 < n_blocks && (!mbar_wait(smem_u32(&sync.pv_done[i]), n & 1) || !scores(n + 2))) code = 61;
                }
            }
            if (code) {
                atomicExch(status, code);
                *(volatile uint32_t*)&sync.failed = 1;
            }
            code = 0;
        }
        __syncwarp();
        if (code && lane == 0) {
            atomicExch(status, code);
            *(volatile uint32_t*)&sync.failed = 1;
        }
    }
    tc_fence_before();
    __syncthreads();
    if (*(volatile uint32_t*)&sync.failed != 0 && tid == 0)
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);               // let copies in flight land
    __syncthreads();
    if (warp == TC_ISSUE) tmem_dealloc(tmem, TC_COLS);
}

// ---- the ranges of a (row, head) joined: a warp each ------------------------------------------------------------------
// J: features a lane takes (lane, lane + 32, ..).  Eight ranges are asked for at once.
template <typename T, int J>
__global__ void __launch_bounds__(128) attention_shared_join_kernel(SharedArgs a) {
    const int row = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (head >= a.n_head) return;
    const int p = position_of(a, row);
    T* const out = (T*)a.out + ((size_t)row * a.n_head + head) * a.D;
    pdl_wait();
    pdl_trigger();
    const int behind = a.behind[row], own = p + 1 - behind;
    if (p < 0) {                                          // padding of a fixed-size batch
        for (int d = lane; d < a.D; d += 32) out[d] = from_float<T>(0.f);
        return;
    }
    const int shared_step = range_keys(behind, a.shared_slots, a.shared_least), own_step = range_keys(own, a.own_slots, OWN_LEAST);
    const int n_shared = (behind + shared_step - 1) / shared_step, n_all = n_shared + (own + own_step - 1) / own_step;
    const size_t base = ((size_t)row * a.n_head + head) * (a.shared_slots + a.own_slots);
    const int skip = a.shared_slots - n_shared;           // slots of shared ranges that this length does not have
    // averages relative to the largest maximum so far
    float top = -INFINITY, total = 0.f, acc[J];
#pragma unroll
    for (int j = 0; j < J; ++j) acc[j] = 0.f;
    for (int i0 = 0; i0 < n_all; i0 += 8) {
        float x[8][J];
        float2 ml[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const bool in = i0 + u < n_all;
            const size_t at = base + i0 + u + (i0 + u < n_shared ? 0 : skip);
            ml[u] = in ? *reinterpret_cast<const float2*>(a.part_ml + at * 2) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int j = 0; j < J; ++j) x[u][j] = in && lane + 32 * j < a.D ? a.part_out[at * a.D + lane + 32 * j] : 0.f;
        }
        float high = top;
#pragma unroll
        for (int u = 0; u < 8; ++u) high = fmaxf(high, ml[u].x);
        const float corr = top == high ? 1.f : exp2f(top - high);
        top = high;
        total *= corr;
#pragma unroll
        for (int j = 0; j < J; ++j) acc[j] *= corr;
#pragma unroll
        for (int u = 0; u < 8; ++u) {                     // ranges in order
            if (ml[u].x == -INFINITY && ml[u].y == 0.f) continue;
            const float w = top == -INFINITY ? 1.f : exp2f(ml[u].x - top);
            total = fmaf(w, ml[u].y, total);
#pragma unroll
            for (int j = 0; j < J; ++j) acc[j] = fmaf(w, x[u][j], acc[j]);
        }
    }
    const float inv = result_of(1.f, top, total);
#pragma unroll
    for (int j = 0; j < J; ++j)
        if (lane + 32 * j < a.D) out[lane + 32 * j] = from_float<T>(acc[j] * inv);
}

int simt_pairs(int pairs) { return pairs <= 8 ? 8 : 16; }

// A kernel that may start while the one in front of it, which is this operator's own, still runs.
template <typename... KArgs>
int launch_behind(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t s, const SharedArgs& a) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "attention (shared): %s", cudaGetErrorString(e));
    MG_CHECK_LAUNCH("attention (shared)");
    return MG_OK;
}

template <typename T>
int launch_join(const SharedArgs& a, cudaStream_t s) {
    const auto kernel = a.D <= 32 ? attention_shared_join_kernel<T, 1> : a.D <= 64 ? attention_shared_join_kernel<T, 2>
                        : a.D <= 128 ? attention_shared_join_kernel<T, 4> : attention_shared_join_kernel<T, 8>;
    return launch_behind(kernel, dim3(a.n, ceil_div(a.n_head, 4)), 128, 0, s, a);
}

template <typename... KArgs>
int launch_ranges(void (*kernel)(KArgs...), int threads, size_t smem, const SharedArgs& a, cudaStream_t s) {
    const cudaError_t e = mg_raise_shared(kernel, smem);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "attention (shared): cannot raise shared memory: %s", cudaGetErrorString(e));
    const long long items = (long long)a.n_groups * a.row_tiles * a.shared_slots + (long long)a.n * a.own_slots - a.first_item;
    const dim3 grid((unsigned)items, a.n_kv_head);
    if (a.first_item > 0) return launch_behind(kernel, grid, threads, smem, s, a);
    const cudaError_t le = mg_launch(kernel, grid, dim3(threads), smem, s, true, a);
    if (le != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "attention (shared): %s", cudaGetErrorString(le));
    MG_CHECK_LAUNCH("attention (shared)");
    return MG_OK;
}

template <int D>
int launch_tc(const SharedArgs& a, int* status, cudaStream_t s) {
    const int box_rows = a.page_tokens < TC_KEYS ? a.page_tokens : TC_KEYS;
    CUtensorMap map_k, map_v;
    int rc = tensor_map(a.k_pages, a.num_pages * a.n_kv_head * a.page_tokens, D, box_rows, &map_k);
    if (rc == MG_OK) rc = tensor_map(a.v_pages, a.num_pages * a.n_kv_head * a.page_tokens, D, box_rows, &map_v);
    if (rc != MG_OK) return rc;
    const cudaError_t e = mg_raise_shared(attention_shared_tc_kernel<D>, TcSizes<D>::SMEM);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "attention (shared): cannot raise shared memory: %s", cudaGetErrorString(e));
    const cudaError_t le = mg_launch(attention_shared_tc_kernel<D>, dim3((unsigned)(a.n_groups * a.row_tiles * a.shared_slots), a.n_kv_head),
                                     dim3(TC_THREADS), TcSizes<D>::SMEM, s, true, a, map_k, map_v, box_rows, status);
    if (le != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "attention (shared, tcgen05): %s", cudaGetErrorString(le));
    MG_CHECK_LAUNCH("attention (shared, tcgen05)");
    return MG_OK;
}

template <typename T, bool VEC>
int launch_simt(const SharedArgs& a, int pairs, cudaStream_t s) {
    const int nq = simt_pairs(pairs);
    const size_t smem = sizeof(float) * ((size_t)a.D * nq + (size_t)BLOCK_KEYS * (2 * a.D + 1 + nq));
    return nq == 8 ? launch_ranges(attention_shared_simt_kernel<T, 8, VEC>, SIMT_THREADS, smem, a, s)
                   : launch_ranges(attention_shared_simt_kernel<T, 16, VEC>, SIMT_THREADS, smem, a, s);
}

constexpr int DIRECT_KEYS = 256, DIRECT_ROWS = 256, TC_LEAST_PAIRS = 32, TC_CTA_KEYS = 1000;

// Head sizes that the kernels of unshared keys take with weights of bfloat16 (attention_decode.cu); others: see FULL.
bool rounded_weights(int d) { return d == 16 || d == 32 || d == 64 || d == 128 || d == 256; }

template <int DP, int NT, bool MANY>
int launch_mma_tiles(const SharedArgs& a, cudaStream_t s) {
    return launch_ranges(rounded_weights(a.D) ? attention_shared_mma_kernel<DP, NT, MANY, false> : attention_shared_mma_kernel<DP, NT, MANY, true>,
                         MMA_THREADS, MmaSizes<DP, NT, MANY>::SMEM, a, s);
}
template <int DP>
int launch_mma(const SharedArgs& a, int pair_tiles, bool many, cudaStream_t s) {
    if constexpr (DP == 128)
        if (pair_tiles == 1 && many) return launch_mma_tiles<DP, 1, true>(a, s);
    if (pair_tiles == 1) return launch_mma_tiles<DP, 1, false>(a, s);
    if constexpr (DP <= 128)
        if (pair_tiles == 2) return launch_mma_tiles<DP, 2, false>(a, s);
    if constexpr (DP <= 64)
        if (pair_tiles == 4) return launch_mma_tiles<DP, 4, false>(a, s);
    return mg_set_error(MG_ERR_ARG, "attention (shared): no kernel for %d tiles of pairs", pair_tiles);
}

int padded_head(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 128 ? 128 : 256; }

// Where the maxima and sums lie behind the averages in the scratch, in floats (pairs of them are read at once).
size_t sums_at(size_t slots, int head_dim) { return (slots * head_dim + 3) / 4 * 4; }

// How a launch is cut.
// (aligned: pages and rows of queries at 16-byte boundaries, and a scale above zero: the tiles take the largest score before they
// scale it)
enum Kind { F32 = 0, BF16_ALIGNED = 1, BF16 = 2 };
struct Cut {
    bool direct;         // a range a row, no groups: one launch
    bool mma, tc;        // the warp-level tensor cores; shared ranges on tcgen05
    int pair_tiles;      // mma: tiles of 8 pairs that a CTA takes at once
    bool many;           // mma: many CTAs of few keys
    int row_tiles;       // CTAs that share the pairs of a group
    int shared_slots, own_slots;      // ranges of shared keys, and of a row's own
    int shared_least;
    int pairs;           // most pairs that a CTA's rows have
    int launches() const { return direct ? 1 : tc ? 3 : 2; }
};
Cut cut(int n_groups, int max_rows, int max_tokens, int max_behind, int n, int n_head, int n_kv_head, int head_dim, int page_tokens,
        int kind) {
    Cut c;
    // So few keys that reading them once a row costs less than a second kernel in bfloat16.  (8 heads of 64, three quarters of the keys
    // shared, in a captured step, two kernels / one, us: 4 rows of 94 keys 6.1 / 4.5, of 256 6.0 / 6.0, of 512 7.0 / 9.0; 64 rows of
    // 128 8.1 / 6.8, of 256 8.2 / 9.6, of 1,024 15.2 / 25.7; 256 rows of 128 22.6 / 15.3, of 256 23.5 / 22.4, of 512 29.2 / 33.6; 512
    // rows of 128 33.4 / 27.5, of 190 34.8 / 33.6, of 256 36.7 / 39.2.  In 32 bits, where one launch costs time: 4 rows of 94 11.2 / 13.2,
    // of 256 11.8 / 26.0; 64 rows of 128 16.8 / 20.9; 256 rows of 128 64 / 69.)
    const long long keys = n_groups == 0 ? max_behind : (long long)max_tokens + max_behind;
    c.direct = keys <= DIRECT_KEYS / 2 || (keys <= DIRECT_KEYS && (n_groups == 0 || n <= DIRECT_ROWS));
    if (c.direct) n_groups = 0;
    const int share = n_head / n_kv_head, pairs = n_groups > 0 ? (max_rows < n ? max_rows : n) * share : share;
    c.mma = kind == BF16_ALIGNED && head_dim % 8 == 0;
    // tcgen05 from 32 pairs on.  (mma.sync / tcgen05, us in a captured step, 2,000 shared tokens: 8 heads of 64, 16 pairs 14.6 / 15.6, 32
    // 23.2 / 16.3 and with 300 tokens 11.4 / 10.1, 128 32.3 / 21.9; 32/8 heads of 128, 16 pairs 20.8 / 17.0 and with 300 tokens
    // 9.3 / 11.1, 32 20.5 / 17.4 and with 300 tokens 10.0 / 11.6, 512 75.9 / 33.6.)
    c.tc = n_groups > 0 && kind == BF16_ALIGNED && (head_dim == 64 || head_dim == 128) && pairs >= TC_LEAST_PAIRS && page_tokens % 8 == 0 &&
           (page_tokens < TC_KEYS ? TC_KEYS % page_tokens == 0 : page_tokens % TC_KEYS == 0) && max_tokens >= TC_KEYS;
    const int most_tiles = head_dim <= 64 ? 4 : head_dim <= 128 ? 2 : 1;      // what the registers hold
    const int mma_pairs = c.tc ? share : pairs;
    c.pair_tiles = mma_pairs <= 8 ? 1 : mma_pairs <= 16 && most_tiles > 1 ? 2 : most_tiles;
    c.row_tiles = ceil_div(pairs, c.tc ? TC_TILES * TC_PAIRS : c.mma ? 8 * c.pair_tiles : simt_pairs(pairs));
    c.shared_least = c.tc ? TC_KEYS : BLOCK_KEYS;
    const long long shared_ctas = (long long)n_groups * c.row_tiles * n_kv_head, own_ctas = (long long)n * n_kv_head;
    const int most_shared = ceil_div(max_tokens > 0 ? max_tokens : 1, c.shared_least), most_own = ceil_div(max_behind, OWN_LEAST);
    // (CTAs of each kind; us in a captured step with one, two and four an SM: 8 x 8 rows of about 1,021 shared tokens, 8 heads of 64
    // 11.7, 12.9, 14.7; 4 rows of 2,000 10.2, 12.2, 12.1; 8 x 8 rows of 1,000, 32/8 heads of 128 26.7, 26.8, 27.1; 2 x 5 rows of 509, 12
    // heads of 64 in 32 bits 19.3, 14.8, 14.8)
    const long long want = 148 * 2;
    long long x = shared_ctas > 0 ? (want + shared_ctas - 1) / shared_ctas : 1;
    if (c.tc) {
        // one CTA an SM: the number of ranges whose rounds of CTAs take the fewest keys, what a CTA costs besides its keys
        // counted as TC_CTA_KEYS of them
        double best = 0.0;
        for (int r = 1; r <= most_shared && r <= 64; ++r) {
            const double cost = (double)((shared_ctas * r + 147) / 148) * ((double)max_tokens / r + TC_CTA_KEYS);
            if (r == 1 || cost < best) { best = cost; x = r; }
        }
    }
    const long long y = (want + own_ctas - 1) / own_ctas;
    c.shared_slots = (int)(x < 1 ? 1 : x > most_shared ? most_shared : x);
    c.own_slots = c.direct ? 1 : (int)(y < 1 ? 1 : y > most_own ? most_own : y);
    // More CTAs than three an SM, none of more than 512 keys.  (Heads of 128, a CTA a row of 8 pairs or fewer, three CTAs an SM / six:
    // 2,048 CTAs of 128 keys 38 / 31 us, 832 of 200 20.5 / 18.1; 832 of 800 37.4 / 40.6, 328 of 865 36 / 44.6.)
    const long long mma_ctas = own_ctas * c.own_slots + (c.tc ? 0 : shared_ctas * c.shared_slots);
    const int range = max(ceil_div(max_behind, c.own_slots), c.tc ? 0 : ceil_div(max_tokens, c.shared_slots));
    c.many = mma_ctas > 148 * 3 && range <= 512;
    c.pairs = pairs;
    return c;
}

}  // namespace

// Floats of scratch that mg_attention_shared() takes for these sizes and bounds.
MG_API long long mg_attention_shared_scratch_floats(int n_groups, int max_rows, int max_tokens, int max_behind, int n, int n_head,
                                                    int n_kv_head, int head_dim, int page_tokens, int kind) {
    if (n_groups < 0 || max_rows <= 0 || n <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || max_behind <= 0 || page_tokens <= 0) return 0;
    const Cut c = cut(n_groups, max_rows, max_tokens, max_behind, n, n_head, n_kv_head, head_dim, page_tokens, kind);
    if (c.direct) return 0;
    const size_t slots = (size_t)n * n_head * (c.shared_slots + c.own_slots);
    return (long long)(sums_at(slots, head_dim) + 2 * slots + n);
}

MG_API int mg_attention_shared_launches(int n_groups, int max_rows, int max_tokens, int max_behind, int n, int n_head, int n_kv_head,
                                        int head_dim, int page_tokens, int kind) {
    if (n <= 0 || max_rows <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || max_behind <= 0 || page_tokens <= 0) return 0;
    return cut(n_groups, max_rows, max_tokens, max_behind, n, n_head, n_kv_head, head_dim, page_tokens, kind).launches();
}

// Attention of n single query tokens, groups of which share their first keys.  q: rows of q_stride elements whose first
// n_head * head_dim are the queries; pages [num_pages, n_kv_head, page_tokens, head_dim]; table [n_requests, max_pages]
// (a page below zero or beyond the pool: its keys are not there); groups [n_groups, 3] ints on the device = (first row,
// rows, shared tokens): rows of different groups are different ones, and the block tables of those of a group's rows that
// see all its shared tokens lead to the same keys and values over them.  max_rows, max_tokens, max_behind: how many rows a group has, how many
// tokens it shares and how many keys a row has besides, at most (bounds that are too low cost time).  A row whose position
// is below zero is padding: its output is zeros.  scratch: mg_attention_shared_scratch_floats() floats, 16-byte aligned,
// that no other launch uses meanwhile.  kind: 0 32-bit, 1 bfloat16 with pages and rows of queries at 16-byte boundaries and a scale
// above zero, 2 other bfloat16.  status: a word that gets a code if a bounded wait runs out.  mg_attention_shared_launches()
// launches.  MG_ERR_UNSUPPORTED for heads of more than 256 features.
MG_API int mg_attention_shared(const void* q, long long q_stride, const void* k_pages, const void* v_pages, const int* table,
                               const int* token_request, const int* positions, const int* groups, int n_groups, int max_rows,
                               int max_tokens, int max_behind, void* out, float* scratch, int n, int n_head, int n_kv_head,
                               int head_dim, int page_tokens, int max_pages, int num_pages, int n_requests, float scale,
                               int kind, int* status, void* stream) {
    const bool is_bf16 = kind != F32;
    if (n == 0) return MG_OK;
    MG_REQUIRE(n > 0 && n_head > 0 && n_kv_head > 0 && head_dim > 0 && page_tokens > 0 && max_pages > 0 && num_pages > 0 && n_requests > 0,
               "attention (shared): bad sizes");
    MG_REQUIRE(n_head % n_kv_head == 0, "attention: n_head %d is not a multiple of n_kv_head %d", n_head, n_kv_head);
    MG_REQUIRE(n_groups >= 0 && (n_groups == 0 || (groups && max_rows > 0 && max_tokens >= 0)) && max_behind > 0 &&
                   max_tokens <= (1 << 30) && max_behind <= (1 << 30),
               "attention (shared): bad groups or bounds");
    MG_REQUIRE(q_stride >= (long long)n_head * head_dim, "attention (shared): rows too narrow");
    MG_REQUIRE((long long)num_pages * n_kv_head * page_tokens < (1ll << 31), "attention (shared): the pool has too many rows");
    if (head_dim > 256 || n_kv_head > 65535)
        return mg_set_error(MG_ERR_UNSUPPORTED, "attention (shared): head_dim %d is more than 256", head_dim);
    SharedArgs a;
    const Cut c = cut(n_groups, max_rows, max_tokens, max_behind, n, n_head, n_kv_head, head_dim, page_tokens, kind);
    a.q = q; a.q_stride = q_stride; a.k_pages = k_pages; a.v_pages = v_pages; a.table = table; a.token_request = token_request;
    a.positions = positions; a.groups = groups; a.out = out;
    a.n_groups = n_groups; a.n = n; a.n_head = n_head; a.n_kv_head = n_kv_head; a.D = head_dim; a.page_tokens = page_tokens;
    a.max_pages = max_pages; a.num_pages = num_pages; a.n_requests = n_requests;
    MG_REQUIRE(c.direct || scratch != nullptr, "attention (shared): no scratch");
    if (c.direct) a.n_groups = n_groups = 0;
    a.direct = c.direct; a.element = is_bf16 ? 2 : 4;
    a.page_shift = (page_tokens & (page_tokens - 1)) == 0 ? __builtin_ctz(page_tokens) : -1;
    a.first_item = 0; a.shared_least = c.shared_least;
    a.row_tiles = c.row_tiles; a.shared_slots = c.shared_slots; a.own_slots = c.own_slots;
    a.scale_log2e = scale * 1.4426950408889634f;
    const size_t slots = (size_t)n * n_head * (c.shared_slots + c.own_slots);
    a.part_out = scratch;
    a.part_ml = scratch + sums_at(slots, head_dim);
    a.behind = (int*)(a.part_ml + 2 * slots);
    const long long items = (long long)n_groups * c.row_tiles * c.shared_slots + (long long)n * c.own_slots;
    MG_REQUIRE(items < (1ll << 31), "attention (shared): too many rows");
    cudaStream_t s = (cudaStream_t)stream;
    int rc;
    MG_REQUIRE(kind != BF16_ALIGNED || (q_stride % 8 == 0 && (((uintptr_t)q | (uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0),
               "attention (shared): rows that are said to be 16-byte aligned and are not");
    MG_REQUIRE(kind != BF16_ALIGNED || scale > 0.f, "attention (shared): a scale that is said to be above zero and is not");
    if (c.tc) {
        rc = head_dim == 64 ? launch_tc<64>(a, status, s) : launch_tc<128>(a, status, s);
        if (rc != MG_OK) return rc;
        a.first_item = n_groups * c.row_tiles * c.shared_slots;         // what is left are the rows' own ranges
    }
    if (c.mma) {
        switch (padded_head(head_dim)) {
            case 32: rc = launch_mma<32>(a, c.pair_tiles, c.many, s); break;
            case 64: rc = launch_mma<64>(a, c.pair_tiles, c.many, s); break;
            case 128: rc = launch_mma<128>(a, c.pair_tiles, c.many, s); break;
            default: rc = launch_mma<256>(a, c.pair_tiles, c.many, s);
        }
    } else {
        rc = is_bf16 ? launch_simt<bf16, false>(a, c.pairs, s)
             : head_dim % 4 == 0 && ((((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) == 0) ? launch_simt<float, true>(a, c.pairs, s)
                                                                                           : launch_simt<float, false>(a, c.pairs, s);
    }
    if (rc != MG_OK || c.direct) return rc;
    return is_bf16 ? launch_join<bf16>(a, s) : launch_join<float>(a, s);
}
