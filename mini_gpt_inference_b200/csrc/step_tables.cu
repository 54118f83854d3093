// Block tables, positions and slot maps of a step, from the lengths of its requests, on the device.
//
// A step's integers (parts/context.py) follow from the requests' pages and two numbers per request: the tokens it has in
// the cache and the tokens it brings.  With starts s_r = sum_{i<r} new_i, token t of request r (s_r <= t < s_r + new_r) has the
// position  before_r + t - s_r  and the cache row  page(position / page size) * page size + position mod page size; a block
// table holds the pages of positions below before_r + new_r and -1 behind them.  Where the lengths live on the device (a
// search that takes its own next tokens), nothing of this needs the host.
//
// Every CTA works the starts out for itself (a prefix sum over some hundred numbers, kept in shared memory) and then takes
// its share of the tokens, each of which finds its request by bisection, and of the tables' cells: one launch, no order
// between the CTAs.
#include "common.cuh"

MG_GUARD_DECLARE(step_tables)

namespace {

constexpr int THREADS = 256, MAX_REQUESTS = 4096, MAX_GROUPS = 8;

struct TableGroup {
    const int* pool;         // [pool rows][width] pages of every request that there is
    int* table;              // [requests][width]
    int* slots;              // [tokens]
    int width, page_tokens;
};

struct TableArgs {
    const int* rows;         // row of the pool of each request, or null: request r has row r
    const int* before;
    const int* fresh;
    int* token_request;
    int* positions;
    int* q_start;
    int* after;
    int n_requests, n_tokens, pool_rows, n_groups;
    TableGroup group[MAX_GROUPS];
};

__global__ void __launch_bounds__(THREADS) step_tables_kernel(const __grid_constant__ TableArgs a) {
    extern __shared__ int starts[];                      // [requests + 1]
    __shared__ int warp_total[THREADS / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();                                          // (nothing overlaps its end: see mg_next_launch_waits)
    // starts: each thread sums a run of requests, the runs' sums are scanned over the CTA
    const int per = (a.n_requests + THREADS - 1) / THREADS, r0 = min(a.n_requests, tid * per), r1 = min(a.n_requests, r0 + per);
    int sum = 0;
    for (int r = r0; r < r1; ++r) sum += max(0, a.fresh[r]);
    int scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, scan, o);
        if (lane >= o) scan += v;
    }
    if (lane == 31) warp_total[warp] = scan;
    __syncthreads();
    int at = scan - sum;
    for (int w = 0; w < warp; ++w) at += warp_total[w];
    for (int r = r0; r < r1; ++r) {
        starts[r] = at;
        if (blockIdx.x == 0) {
            a.q_start[r] = at;
            a.after[r] = a.before[r] + max(0, a.fresh[r]);
        }
        at += max(0, a.fresh[r]);
    }
    if (tid == THREADS - 1) starts[a.n_requests] = at;
    __syncthreads();

    const int total = starts[a.n_requests], step = gridDim.x * THREADS;
    for (int t = blockIdx.x * THREADS + tid; t < a.n_tokens; t += step) {
        int lo = 0, hi = a.n_requests;                   // the last request that starts at or before t and brings tokens
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (starts[mid] <= t) lo = mid; else hi = mid;
        }
        const bool real = t < total;
        const int position = real ? a.before[lo] + t - starts[lo] : -1;
        a.token_request[t] = real ? lo : 0;
        a.positions[t] = position;
        int row = real ? (a.rows ? a.rows[lo] : lo) : 0;
        const bool known = real && position >= 0 && row >= 0 && row < a.pool_rows;
        if (real) (void)MG_GUARDED(step_tables, MG_GUARD_ROW, row, a.pool_rows);
#pragma unroll
        for (int g = 0; g < MAX_GROUPS; ++g) {
            if (g >= a.n_groups) break;
            const int column = position / a.group[g].page_tokens;
            int slot = -1;
            if (known && column < a.group[g].width) {
                const int page = a.group[g].pool[(size_t)row * a.group[g].width + column];
                if (page >= 0) slot = page * a.group[g].page_tokens + position - column * a.group[g].page_tokens;
            } else if (known) {
                (void)MG_GUARDED(step_tables, MG_GUARD_POSITION, column, a.group[g].width);
            }
            a.group[g].slots[t] = slot;
        }
    }
#pragma unroll
    for (int g = 0; g < MAX_GROUPS; ++g) {
        if (g >= a.n_groups) break;
        const TableGroup& p = a.group[g];
        for (int r = blockIdx.x; r < a.n_requests; r += gridDim.x) {
            const int row = a.rows ? a.rows[r] : r, end = a.before[r] + max(0, a.fresh[r]);
            const int held = row >= 0 && row < a.pool_rows && end > 0 ? (end + p.page_tokens - 1) / p.page_tokens : 0;
            for (int c = tid; c < p.width; c += THREADS)
                p.table[(size_t)r * p.width + c] = c < held ? p.pool[(size_t)row * p.width + c] : -1;
        }
    }
}

}  // namespace

// rows (or null), before, fresh: [n_requests] ints on the device.  groups: per group of n_groups (at most 8) five numbers: the
// addresses of its pages [pool_rows, width] (below zero: none), of the block tables [n_requests, width] and of the cache rows
// [n_tokens] to be written, width, and tokens of a page.  Token rows behind the last request's are padding: position and cache
// row -1, request 0.  A number of new tokens below zero counts as none.
// after: [n_requests], before + fresh.
MG_API int mg_step_tables(const int* rows, const int* before, const int* fresh, int* token_request, int* positions, int* q_start,
                          int* after, int n_requests, int n_tokens, int pool_rows, int n_groups, const long long* groups, void* stream) {
    if (n_requests == 0 && n_tokens == 0) return MG_OK;
    MG_REQUIRE(n_requests > 0 && n_tokens >= 0 && pool_rows > 0 && n_groups >= 0, "step_tables: bad sizes");
    MG_REQUIRE(n_requests <= MAX_REQUESTS && n_groups <= MAX_GROUPS, "step_tables: at most %d requests and %d groups", MAX_REQUESTS, MAX_GROUPS);
    TableArgs a = {};
    a.rows = rows; a.before = before; a.fresh = fresh; a.token_request = token_request; a.positions = positions; a.q_start = q_start; a.after = after;
    a.n_requests = n_requests; a.n_tokens = n_tokens; a.pool_rows = pool_rows; a.n_groups = n_groups;
    for (int g = 0; g < n_groups; ++g) {
        const long long* z = groups + 5 * g;
        MG_REQUIRE(z[3] > 0 && z[3] < (1ll << 31) && z[4] > 0 && z[4] < (1ll << 31), "step_tables: bad page sizes");
        a.group[g] = {(const int*)z[0], (int*)z[1], (int*)z[2], (int)z[3], (int)z[4]};
    }
    int ctas = ceil_div(n_tokens, THREADS) > n_requests ? ceil_div(n_tokens, THREADS) : n_requests;
    if (ctas > 296) ctas = 296;
    const cudaError_t e = mg_launch(step_tables_kernel, dim3(ctas), dim3(THREADS), sizeof(int) * (n_requests + 1), (cudaStream_t)stream,
                                    true, a);
    if (e != cudaSuccess) return mg_set_error(MG_ERR_CUDA, "step_tables: %s", cudaGetErrorString(e));
    MG_CHECK_LAUNCH("step_tables");
    mg_next_launch_waits();                              // (kernels read these integers before they wait for what is in front of them)
    return MG_OK;
}
