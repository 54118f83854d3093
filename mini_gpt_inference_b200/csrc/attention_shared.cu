// Attention of single query tokens over the paged cache where groups of tokens share their first keys: the beams of a
// search, the samples of one prompt.
//
// A row's result is the softmax average over the keys 0 .. its position, as in the other attention kernels; what differs is
// how often the keys are read.  Where every row reads all of its keys, a prompt of P tokens continued B times is read B
// times.  Here the keys are cut into ranges of two kinds: those of the P tokens that a group's rows share, read once for
// all (row, head) pairs of the group and key/value head, and those behind them, read for their own row.  A range leaves
// per (row, head) its unnormalised average acc, its maximum m (of the scores times log2 e) and its sum l, and a second
// kernel joins them:  M = max m_i,  out = sum 2^(m_i - M) acc_i / sum 2^(m_i - M) l_i.
//
// How many ranges there are is the host's choice, from bounds on the lengths that it knows when it launches (a captured
// step has its grid for good); where the ranges lie is worked out on the device from the lengths as they are: a length is
// cut into as many ranges as there are, of at least a fixed number of keys, so bounds that are too low cost time only.  The
// same holds for the rows of a group.  A row that stands in front of the end of its group's shared tokens reads all its
// keys for itself, and so does one that belongs to no group.
#include <math.h>

#include "common.cuh"

MG_GUARD_DECLARE(attention_shared)

namespace {

constexpr int BLOCK_KEYS = 64;         // ranges are cut at multiples of this many keys

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
    int n_groups, n, n_head, n_kv_head, D, page_tokens, max_pages, num_pages, n_requests;
    int row_tiles;                     // CTAs that share the (row, head) pairs of a group
    int shared_slots, own_slots;       // ranges of the shared keys, and of a row's own
    float scale_log2e;
};

// Keys of one range when `keys` of them are cut into at most `slots`, each of at least `least` keys.
__host__ __device__ __forceinline__ int range_keys(int keys, int slots, int least) {
    const int even = (keys + slots - 1) / slots;
    const int whole = (even + BLOCK_KEYS - 1) / BLOCK_KEYS * BLOCK_KEYS;
    return whole < least ? least : whole;
}

constexpr int SHARED_LEAST = 64, OWN_LEAST = 64;

// The shared tokens of the group that `row` belongs to (0: none), by all threads of a CTA; `hold` is a word of shared memory.
__device__ __forceinline__ int group_tokens(const SharedArgs& a, int row, int* hold) {
    if (threadIdx.x == 0) *hold = 0;
    __syncthreads();
    for (int g = threadIdx.x; g < a.n_groups; g += blockDim.x) {
        const int first = a.groups[3 * g], rows = a.groups[3 * g + 1];
        if (row >= first && row - first < rows) *hold = a.groups[3 * g + 2];
    }
    __syncthreads();
    return *hold;
}

// ---- any head size, either type: 16 (row, head) pairs and 64 keys at a time, in 32-bit arithmetic ------------------------
constexpr int SIMT_THREADS = 128, SIMT_QUERIES = 16;

__host__ __device__ constexpr int simt_lanes(int d) { return d > 64 ? 128 : d > 32 ? 64 : 32; }     // threads across the features

template <typename T>
__global__ void __launch_bounds__(SIMT_THREADS) attention_shared_simt_kernel(SharedArgs a) {
    extern __shared__ float smem[];
    __shared__ int krow[BLOCK_KEYS], q_token[SIMT_QUERIES], q_head[SIMT_QUERIES], hold;
    __shared__ float q_max[SIMT_QUERIES], q_sum[SIMT_QUERIES], q_corr[SIMT_QUERIES];
    const int tid = threadIdx.x, D = a.D, kv_head = blockIdx.y, share = a.n_head / a.n_kv_head;
    float* q_s = smem;                                   // [D][16]
    float* k_s = q_s + D * SIMT_QUERIES;                 // [64][D + 1]
    float* p_s = k_s + BLOCK_KEYS * (D + 1);             // [64][16]
    const int lanes = simt_lanes(D), dl = tid % lanes, ks = tid / lanes, key_parts = SIMT_THREADS / lanes;

    // which queries and which keys
    const int shared_items = a.n_groups * a.row_tiles * a.shared_slots;
    int item = blockIdx.x, first_row, rows, key0, key1, slot, tile, tiles;
    const bool shared = item < shared_items;
    if (shared) {
        slot = item % a.shared_slots;
        item /= a.shared_slots;
        tile = item % a.row_tiles;
        tiles = a.row_tiles;
        const int g = item / a.row_tiles;
        first_row = a.groups[3 * g];
        rows = a.groups[3 * g + 1];
        const int keys = a.groups[3 * g + 2], step = range_keys(keys, a.shared_slots, SHARED_LEAST);
        key0 = slot * step;
        key1 = min(keys, key0 + step);
        if (first_row < 0 || rows <= 0 || first_row >= a.n) return;
        rows = min(rows, a.n - first_row);
    } else {
        item -= shared_items;
        slot = item % a.own_slots;
        first_row = item / a.own_slots;
        rows = 1;
        tile = 0;
        tiles = 1;
        const int p = a.positions[first_row];
        int behind = group_tokens(a, first_row, &hold);
        if (behind > p + 1) behind = 0;
        const int step = range_keys(p + 1 - behind, a.own_slots, OWN_LEAST);
        key0 = behind + slot * step;
        key1 = min(p + 1, key0 + step);
        slot += a.shared_slots;
    }
    if (key0 >= key1) return;
    int request = a.token_request[first_row];
    if (!MG_GUARDED(attention_shared, MG_GUARD_REQUEST, request, a.n_requests)) request = 0;
    const int* table = a.table + (size_t)request * a.max_pages;
    const int shared_keys = shared ? a.groups[3 * (blockIdx.x / (a.shared_slots * a.row_tiles)) + 2] : 0;

    for (int q0 = tile * SIMT_QUERIES; q0 < rows * share; q0 += tiles * SIMT_QUERIES) {
        __syncthreads();
        if (tid < SIMT_QUERIES) {
            const int j = q0 + tid, row = first_row + j / share;
            // (a row that does not see all the shared keys is no row of this range)
            const bool in = j < rows * share && (!shared || a.positions[row] + 1 >= shared_keys);
            q_token[tid] = in ? row : -1;
            q_head[tid] = kv_head * share + j % share;
            q_max[tid] = -INFINITY;
            q_sum[tid] = 0.f;
        }
        __syncthreads();
        for (int i = tid; i < SIMT_QUERIES * D; i += SIMT_THREADS) {
            const int j = i / D, d = i - j * D;
            q_s[d * SIMT_QUERIES + j] =
                q_token[j] < 0 ? 0.f : to_float(((const T*)a.q)[q_token[j] * a.q_stride + (size_t)q_head[j] * D + d]) * a.scale_log2e;
        }
        float acc[2][SIMT_QUERIES];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < SIMT_QUERIES; ++j) acc[i][j] = 0.f;
        for (int b0 = key0; b0 < key1; b0 += BLOCK_KEYS) {
            __syncthreads();
            if (tid < BLOCK_KEYS) {
                const int pos = b0 + tid, pi = pos / a.page_tokens;
                int page = pos < key1 && pi < a.max_pages ? table[pi] : -1;
                if (page >= 0 && !MG_GUARDED(attention_shared, MG_GUARD_PAGE, page, a.num_pages)) page = -1;
                if (page >= a.num_pages) page = -1;      // a key without a page is not there
                krow[tid] = page < 0 ? -1 : pos - pi * a.page_tokens;
                if (page >= 0) krow[tid] += (page * a.n_kv_head + kv_head) * a.page_tokens;
            }
            __syncthreads();
            for (int i = tid; i < BLOCK_KEYS * D; i += SIMT_THREADS) {
                const int r = i / D, d = i - r * D;
                k_s[r * (D + 1) + d] = krow[r] < 0 ? 0.f : to_float(((const T*)a.k_pages)[(size_t)krow[r] * D + d]);
            }
            __syncthreads();
            {
                const int key = tid & (BLOCK_KEYS - 1), j0 = (tid / BLOCK_KEYS) * 8;
                float s[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) s[j] = 0.f;
                for (int d = 0; d < D; ++d) {
                    const float k = k_s[key * (D + 1) + d];
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[j] = fmaf(k, q_s[d * SIMT_QUERIES + j0 + j], s[j]);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) p_s[key * SIMT_QUERIES + j0 + j] = krow[key] < 0 ? -INFINITY : s[j];
            }
            __syncthreads();
            {
                const int j = tid >> 3, part = tid & 7;              // eight neighbouring threads a query
                float m = -INFINITY;
                for (int k = part; k < BLOCK_KEYS; k += 8) m = fmaxf(m, p_s[k * SIMT_QUERIES + j]);
#pragma unroll
                for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                const float before = q_max[j], top = fmaxf(before, m);
                float sum = 0.f;
                for (int k = part; k < BLOCK_KEYS; k += 8) {
                    const float e = top == -INFINITY ? 0.f : exp2f(p_s[k * SIMT_QUERIES + j] - top);
                    p_s[k * SIMT_QUERIES + j] = e;
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
                for (int j = 0; j < SIMT_QUERIES; ++j) acc[i][j] *= q_corr[j];
            for (int k = ks; k < BLOCK_KEYS; k += key_parts) {
                if (krow[k] < 0) continue;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int d = dl + i * SIMT_THREADS;
                    if (d >= D) break;
                    const float v = to_float(((const T*)a.v_pages)[(size_t)krow[k] * D + d]);
#pragma unroll
                    for (int j = 0; j < SIMT_QUERIES; ++j) acc[i][j] = fmaf(p_s[k * SIMT_QUERIES + j], v, acc[i][j]);
                }
            }
        }
        // the threads that shared the keys of a feature meet (the key tile is free: scratch)
        if (key_parts > 1) {
            __syncthreads();
            if (ks > 0 && dl < D)
#pragma unroll
                for (int j = 0; j < SIMT_QUERIES; ++j) k_s[((ks - 1) * SIMT_QUERIES + j) * D + dl] = acc[0][j];
            __syncthreads();
            if (ks == 0 && dl < D)
                for (int other = 0; other < key_parts - 1; ++other)
#pragma unroll
                    for (int j = 0; j < SIMT_QUERIES; ++j) acc[0][j] += k_s[(other * SIMT_QUERIES + j) * D + dl];
        }
        const int slots = a.shared_slots + a.own_slots;
        if (ks == 0)
#pragma unroll
            for (int j = 0; j < SIMT_QUERIES; ++j) {
                if (q_token[j] < 0) continue;
                const size_t at = ((size_t)q_token[j] * a.n_head + q_head[j]) * slots + slot;
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (dl + i * SIMT_THREADS < D) a.part_out[at * D + dl + i * SIMT_THREADS] = acc[i][j];
                if (dl == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(q_max[j], q_sum[j]);
            }
    }
}

// ---- the ranges of a (row, head) joined: a warp each ------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(128) attention_shared_join_kernel(SharedArgs a) {
    __shared__ int hold;
    const int row = blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int p = a.positions[row];
    int behind = group_tokens(a, row, &hold);
    if (behind > p + 1) behind = 0;
    if (head >= a.n_head) return;
    T* out = (T*)a.out + ((size_t)row * a.n_head + head) * a.D;
    if (p < 0) {                                          // padding of a fixed-size batch
        for (int d = lane; d < a.D; d += 32) out[d] = from_float<T>(0.f);
        return;
    }
    const int shared_step = range_keys(behind, a.shared_slots, SHARED_LEAST), own = p + 1 - behind;
    const int own_step = range_keys(own, a.own_slots, OWN_LEAST);
    const int n_shared = (behind + shared_step - 1) / shared_step, n_all = n_shared + (own + own_step - 1) / own_step;
    const size_t base = ((size_t)row * a.n_head + head) * (a.shared_slots + a.own_slots);
    const int skip = a.shared_slots - n_shared;           // slots of shared ranges that this length does not have
    float top = -INFINITY;
    for (int i = lane; i < n_all; i += 32) top = fmaxf(top, a.part_ml[(base + i + (i < n_shared ? 0 : skip)) * 2]);
    top = warp_max(top);
    float acc[8], total = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = 0.f;
    for (int i = 0; i < n_all; ++i) {
        const size_t at = base + i + (i < n_shared ? 0 : skip);
        const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2);
        const float w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
        total = fmaf(w, ml.y, total);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 32 * j < a.D) acc[j] = fmaf(w, a.part_out[at * a.D + lane + 32 * j], acc[j]);
    }
    const float inv = total > 0.f ? 1.0f / total : 0.f;   // (no key has a page: zeros)
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (lane + 32 * j < a.D) out[lane + 32 * j] = from_float<T>(acc[j] * inv);
}

template <typename T>
int launch_simt(const SharedArgs& a, cudaStream_t s) {
    const size_t smem = sizeof(float) * ((size_t)a.D * SIMT_QUERIES + (size_t)BLOCK_KEYS * (a.D + 1) + BLOCK_KEYS * SIMT_QUERIES);
    const cudaError_t e = mg_raise_shared(attention_shared_simt_kernel<T>, smem);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "attention (shared): cannot raise shared memory: %s", cudaGetErrorString(e));
    const long long items = (long long)a.n_groups * a.row_tiles * a.shared_slots + (long long)a.n * a.own_slots;
    attention_shared_simt_kernel<T><<<dim3((unsigned)items, a.n_kv_head), SIMT_THREADS, smem, s>>>(a);
    MG_CHECK_LAUNCH("attention (shared)");
    attention_shared_join_kernel<T><<<dim3(a.n, ceil_div(a.n_head, 4)), 128, 0, s>>>(a);
    MG_CHECK_LAUNCH("attention (shared, join)");
    return MG_OK;
}

// How a launch is cut: [0] CTAs that share the pairs of a group, [1] ranges of shared keys, [2] ranges of own keys.
void cut(int n_groups, int max_rows, int max_tokens, int max_behind, int n, int n_head, int n_kv_head, int* out) {
    const int share = n_head / n_kv_head;
    out[0] = ceil_div(max_rows * share, SIMT_QUERIES);
    const long long shared_ctas = (long long)n_groups * out[0] * n_kv_head, own_ctas = (long long)n * n_kv_head;
    const int most_shared = ceil_div(max_tokens > 0 ? max_tokens : 1, SHARED_LEAST), most_own = ceil_div(max_behind, OWN_LEAST);
    const long long want = 148 * 4;
    long long a = shared_ctas > 0 ? (want + shared_ctas - 1) / shared_ctas : 1, b = (want + own_ctas - 1) / own_ctas;
    out[1] = (int)(a < 1 ? 1 : a > most_shared ? most_shared : a);
    out[2] = (int)(b < 1 ? 1 : b > most_own ? most_own : b);
}

}  // namespace

// Floats of scratch that mg_attention_shared() takes for these sizes and bounds.
MG_API long long mg_attention_shared_scratch_floats(int n_groups, int max_rows, int max_tokens, int max_behind, int n, int n_head,
                                                    int n_kv_head, int head_dim) {
    if (n_groups < 0 || max_rows <= 0 || n <= 0 || n_head <= 0 || n_kv_head <= 0 || n_head % n_kv_head != 0 || max_behind <= 0) return 0;
    int c[3];
    cut(n_groups, max_rows, max_tokens, max_behind, n, n_head, n_kv_head, c);
    return (long long)n * n_head * (c[1] + c[2]) * (head_dim + 2);
}

// Attention of n single query tokens, groups of which share their first keys.  q: rows of q_stride elements whose first
// n_head * head_dim are the queries; pages [num_pages, n_kv_head, page_tokens, head_dim]; table [n_requests, max_pages]
// (a page below zero or beyond the pool: its keys are not there); groups [n_groups, 3] ints on the device = (first row,
// rows, shared tokens): rows of different groups are different ones, and the block tables of a group's rows lead to the
// same keys and values over the shared tokens.  max_rows, max_tokens, max_behind: how many rows a group has, how many
// tokens it shares and how many keys a row has besides, at most (bounds that are too low cost time).  A row whose position
// is below zero is padding: its output is zeros.  scratch: mg_attention_shared_scratch_floats() floats, 16-byte aligned,
// that no other launch uses meanwhile.  Two launches.  MG_ERR_UNSUPPORTED for heads of more than 256 features.
MG_API int mg_attention_shared(const void* q, long long q_stride, const void* k_pages, const void* v_pages, const int* table,
                               const int* token_request, const int* positions, const int* groups, int n_groups, int max_rows,
                               int max_tokens, int max_behind, void* out, float* scratch, int n, int n_head, int n_kv_head,
                               int head_dim, int page_tokens, int max_pages, int num_pages, int n_requests, float scale,
                               int is_bf16, void* stream) {
    if (n == 0) return MG_OK;
    MG_REQUIRE(n > 0 && n_head > 0 && n_kv_head > 0 && head_dim > 0 && page_tokens > 0 && max_pages > 0 && num_pages > 0 && n_requests > 0,
               "attention (shared): bad sizes");
    MG_REQUIRE(n_head % n_kv_head == 0, "attention: n_head %d is not a multiple of n_kv_head %d", n_head, n_kv_head);
    MG_REQUIRE(n_groups >= 0 && (n_groups == 0 || (groups && max_rows > 0 && max_tokens >= 0)) && max_behind > 0,
               "attention (shared): bad groups or bounds");
    MG_REQUIRE(scratch != nullptr && q_stride >= (long long)n_head * head_dim, "attention (shared): no scratch, or rows too narrow");
    MG_REQUIRE((long long)num_pages * n_kv_head * page_tokens < (1ll << 31), "attention (shared): the pool has too many rows");
    if (head_dim > 256 || n_kv_head > 65535)
        return mg_set_error(MG_ERR_UNSUPPORTED, "attention (shared): head_dim %d is more than 256", head_dim);
    SharedArgs a;
    int c[3];
    cut(n_groups, max_rows, max_tokens, max_behind, n, n_head, n_kv_head, c);
    a.q = q; a.q_stride = q_stride; a.k_pages = k_pages; a.v_pages = v_pages; a.table = table; a.token_request = token_request;
    a.positions = positions; a.groups = groups; a.out = out;
    a.n_groups = n_groups; a.n = n; a.n_head = n_head; a.n_kv_head = n_kv_head; a.D = head_dim; a.page_tokens = page_tokens;
    a.max_pages = max_pages; a.num_pages = num_pages; a.n_requests = n_requests;
    a.row_tiles = c[0]; a.shared_slots = c[1]; a.own_slots = c[2];
    a.scale_log2e = scale * 1.4426950408889634f;
    const size_t slots = (size_t)n * n_head * (c[1] + c[2]);
    a.part_ml = scratch;
    a.part_out = scratch + 2 * slots;
    const long long items = (long long)n_groups * c[0] * c[1] + (long long)n * c[2];
    MG_REQUIRE(items < (1ll << 31), "attention (shared): too many rows");
    return is_bf16 ? launch_simt<bf16>(a, (cudaStream_t)stream) : launch_simt<float>(a, (cudaStream_t)stream);
}
