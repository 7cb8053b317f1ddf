// Block tables and slot maps built on the device from request lengths: the
// growth of a batch by given numbers of tokens (blocks popped from a stack, a
// slot for every new token), and its cut back to given lengths (blocks pushed
// again).
//
// One launch each. Every workgroup scans the batch's lengths for itself (at most
// 4,096 requests: 16 per thread, then a scan over the workgroup), which costs
// less than a launch that hands the sums over, and does its share of the rows,
// table entries or returned blocks from them. The state that the scan reads
// (lengths, held blocks, the stack's count) is replaced by the workgroup that
// finishes last: it finds out by a counter that it leaves at zero again, and
// since the others only read that state and nothing is handed over, no fence is
// needed. What is written besides -- rows, fresh table entries, stack entries
// above the count -- is read by no workgroup of the launch.
#include <algorithm>
#include <climits>

#include "mf_common.h"

namespace mf {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxRequests = 4096;
constexpr int kPerThread = kMaxRequests / kThreads;
constexpr int kRowsPerThread = 8;

struct TableArgs {
    int32_t* tables;
    int64_t table_stride;
    int max_blocks;
    int32_t* lens;
    int32_t* held;
    int32_t* free_blocks;
    int64_t free_capacity;
    int32_t* free_count;
    const int32_t* want;  // extend: new tokens; truncate: lengths left
    int num_requests;
    int block_size;
    int64_t max_rows;
    const int32_t* rows;  // extend: (requests, rows_stride) row of each new token, or none
    int64_t rows_stride;
    int rows_width;
    int64_t* slot_mapping;
    int64_t* positions;
    int32_t* cu_seqlens;
    int32_t* kv_lens;
    int32_t* refused;
    uint32_t* arrivals;
};

// Exclusive sums over the workgroup of each thread's v, and the total.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& total) {
    __shared__ int64_t waves[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(incl, o, 64);
        if (lane >= o) incl += up;
    }
    __syncthreads();  // an earlier call's sums have been read
    if (lane == 63) waves[wave] = incl;
    __syncthreads();
    int64_t base = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) base += waves[w];
        total += waves[w];
    }
    return base + incl - v;
}

// Whether this workgroup is the launch's last one to get here; all of its
// threads have then read what they needed of the state.
__device__ __forceinline__ bool last_to_finish(uint32_t* arrivals) {
    __shared__ bool last;
    __syncthreads();
    if (threadIdx.x == 0) {
        last = atomicAdd(arrivals, 1u) == gridDim.x - 1;
        if (last) *arrivals = 0;
    }
    __syncthreads();
    return last;
}

__device__ __forceinline__ int clamp_count(int64_t x) { return (int)min(x, (int64_t)INT_MAX); }

__global__ __launch_bounds__(kThreads) void fill_rows_kernel(int64_t* slots, int64_t* positions, int64_t n) {
    const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    for (int64_t i = at; i < n; i += (int64_t)gridDim.x * kThreads) {
        slots[i] = -1;
        positions[i] = 0;
    }
}

// What one request holds and gets.
struct Request {
    int len, held, grow;
    int64_t n;
    bool fits;
};

__device__ __forceinline__ Request load_request(const TableArgs& a, int s) {
    Request r;
    r.len = max(a.lens[s], 0);
    r.held = min(max(a.held[s], 0), a.max_blocks);
    r.n = max(a.want[s], 0);
    const int64_t need = ((int64_t)r.len + r.n + a.block_size - 1) / a.block_size;
    r.fits = need <= a.max_blocks && (a.rows == nullptr || r.n <= a.rows_width);
    r.grow = r.fits ? (int)max(need - r.held, (int64_t)0) : 0;
    return r;
}

// LDS: the row each request starts at, and the blocks taken before it (-1: the
// request is refused).
__global__ __launch_bounds__(kThreads) void extend_kernel(TableArgs a) {
    __shared__ int cu[kMaxRequests + 1];
    __shared__ int taken[kMaxRequests];
    const int B = a.num_requests;
    const int per = (B + kThreads - 1) / kThreads;
    const int s0 = min((int)threadIdx.x * per, B), s1 = min(s0 + per, B);
    const int count = min(max((int64_t)*a.free_count, (int64_t)0), a.free_capacity);

    // ---- rows, then (those past max_rows left out) blocks
    int64_t rows = 0, total_rows;
    for (int s = s0; s < s1; ++s) rows += max(a.want[s], 0);
    int64_t row = block_scan(rows, total_rows);
    int64_t blocks = 0, total_blocks;
    for (int s = s0; s < s1; ++s) {
        const Request r = load_request(a, s);
        cu[s] = clamp_count(row);
        row += r.n;
        if (row <= a.max_rows) blocks += r.grow;
    }
    if (threadIdx.x == kThreads - 1) cu[B] = clamp_count(total_rows);
    int64_t run = block_scan(blocks, total_blocks);
    row -= rows;
    int refused = 0;
    for (int s = s0; s < s1; ++s) {
        const Request r = load_request(a, s);
        row += r.n;
        const bool fits = r.fits && row <= a.max_rows;
        const int grow = fits ? r.grow : 0;
        run += grow;
        const bool served = fits && (grow == 0 || run <= count);
        taken[s] = served ? (int)(run - grow) : -1;
        refused += !served;
    }
    int64_t all_refused;
    block_scan(refused, all_refused);  // (and a barrier: cu and taken are whole)
    __syncthreads();

    // ---- this workgroup's share of the new tokens' rows
    auto block_of = [&](const int32_t* trow, int held, int base, int j) -> int {
        return j < held ? trow[j] : a.free_blocks[count - 1 - (base + j - held)];
    };
    if (a.rows == nullptr) {
        const int64_t per_wg = (int64_t)kThreads * kRowsPerThread;
        for (int64_t first = (int64_t)blockIdx.x * per_wg; first < a.max_rows; first += (int64_t)gridDim.x * per_wg) {
#pragma unroll 1
            for (int i = 0; i < kRowsPerThread; ++i) {
                const int64_t r = first + (int64_t)i * kThreads + threadIdx.x;
                if (r >= a.max_rows) break;
                int64_t slot = -1, pos = 0;
                if (r < cu[B]) {
                    int lo = 0, hi = B - 1;  // the last request that starts at or before r
                    while (lo < hi) {
                        const int mid = (lo + hi + 1) >> 1;
                        if (cu[mid] <= r) lo = mid;
                        else hi = mid - 1;
                    }
                    pos = max(a.lens[lo], 0) + (r - cu[lo]);
                    if (taken[lo] >= 0) {
                        const int j = (int)(pos / a.block_size);
                        const int held = min(max(a.held[lo], 0), a.max_blocks);
                        const int block = block_of(a.tables + (int64_t)lo * a.table_stride, held, taken[lo], j);
                        slot = (int64_t)block * a.block_size + pos % a.block_size;
                    }
                }
                a.slot_mapping[r] = slot;
                a.positions[r] = pos;
            }
        }
    }

    // ---- its share of the requests: fresh table entries, and rows given by number
    for (int s = (int)blockIdx.x; s < B; s += (int)gridDim.x) {
        if (taken[s] < 0) continue;
        const Request r = load_request(a, s);
        int32_t* trow = a.tables + (int64_t)s * a.table_stride;
        for (int j = (int)threadIdx.x; j < r.grow; j += kThreads)
            trow[r.held + j] = a.free_blocks[count - 1 - (taken[s] + j)];
        if (a.rows != nullptr) {
            for (int j = (int)threadIdx.x; j < (int)r.n; j += kThreads) {
                const int out = a.rows[(int64_t)s * a.rows_stride + j];
                if (out < 0 || out >= a.max_rows) continue;
                const int64_t pos = (int64_t)r.len + j;
                const int block = block_of(trow, r.held, taken[s], (int)(pos / a.block_size));
                a.slot_mapping[out] = (int64_t)block * a.block_size + pos % a.block_size;
                a.positions[out] = pos;
            }
        }
    }
    if (blockIdx.x == 0) {
        for (int s = (int)threadIdx.x; s <= B; s += kThreads) a.cu_seqlens[s] = cu[s];
        if (threadIdx.x == 0) *a.refused = (int)all_refused;
    }

    // ---- the new state
    if (!last_to_finish(a.arrivals)) return;
    int64_t used = 0, total_used;
    for (int s = s0; s < s1; ++s) {
        const Request r = load_request(a, s);
        const bool served = taken[s] >= 0;
        const int len = served ? r.len + (int)r.n : r.len;
        a.lens[s] = len;
        a.kv_lens[s] = len;
        a.held[s] = r.held + (served ? r.grow : 0);
        used += served ? r.grow : 0;
    }
    block_scan(used, total_used);
    if (threadIdx.x == 0) *a.free_count = count - (int)total_used;
}

__global__ __launch_bounds__(kThreads) void truncate_kernel(TableArgs a) {
    __shared__ int before[kMaxRequests];  // blocks that earlier requests give back
    const int B = a.num_requests;
    const int per = (B + kThreads - 1) / kThreads;
    const int s0 = min((int)threadIdx.x * per, B), s1 = min(s0 + per, B);
    const int64_t count = min(max((int64_t)*a.free_count, (int64_t)0), a.free_capacity);
    auto left_of = [&](int s) { return min(max(a.want[s], 0), max(a.lens[s], 0)); };
    auto kept_of = [&](int s) { return (int)(((int64_t)left_of(s) + a.block_size - 1) / a.block_size); };
    auto held_of = [&](int s) { return min(max(a.held[s], 0), a.max_blocks); };
    int64_t back = 0, total;
    for (int s = s0; s < s1; ++s) back += max(held_of(s) - kept_of(s), 0);
    int64_t run = block_scan(back, total);
    for (int s = s0; s < s1; ++s) {
        before[s] = (int)run;
        run += max(held_of(s) - kept_of(s), 0);
    }
    __syncthreads();
    // the last block taken by the last request that grew lies on top again
    for (int s = (int)blockIdx.x; s < B; s += (int)gridDim.x) {
        const int kept = kept_of(s), held = held_of(s);
        int32_t* trow = a.tables + (int64_t)s * a.table_stride;
        for (int j = kept + (int)threadIdx.x; j < held; j += kThreads) {
            const int64_t place = count + total - 1 - (before[s] + j - kept);
            if (place < a.free_capacity) a.free_blocks[place] = trow[j];
            trow[j] = 0;
        }
    }
    if (!last_to_finish(a.arrivals)) return;
    for (int s = s0; s < s1; ++s) {
        const int left = left_of(s), kept = kept_of(s), held = held_of(s);
        a.lens[s] = left;
        a.held[s] = min(held, kept);
    }
    if (threadIdx.x == 0) *a.free_count = (int)min(count + total, a.free_capacity);
}

int check_tables(const TableArgs& a) {
    if (a.num_requests < 0 || a.num_requests > kMaxRequests || a.block_size <= 0 || a.max_blocks < 0 ||
        a.table_stride < a.max_blocks || a.free_capacity < 0 || a.free_capacity > INT_MAX || a.max_rows < 0 ||
        a.max_rows > INT_MAX || !a.free_count || !a.arrivals)
        return MF_ERR_ARG;
    if (a.num_requests > 0 && (!a.lens || !a.held || !a.want)) return MF_ERR_ARG;
    if ((int64_t)a.num_requests * a.max_blocks > 0 && !a.tables) return MF_ERR_ARG;
    if (a.free_capacity > 0 && !a.free_blocks) return MF_ERR_ARG;
    return MF_OK;
}

}  // namespace
}  // namespace mf

extern "C" int mf_tables_extend(int32_t* tables, int64_t table_stride, int max_blocks, int32_t* lens, int32_t* held,
                                int32_t* free_blocks, int64_t free_capacity, int32_t* free_count,
                                const int32_t* new_tokens, int num_requests, int block_size, int64_t max_rows,
                                const int32_t* rows, int64_t rows_stride, int rows_width, int64_t* slot_mapping,
                                int64_t* positions, int32_t* cu_seqlens, int32_t* kv_lens, int32_t* refused,
                                uint32_t* arrivals, mf_stream_t stream) {
    using namespace mf;
    TableArgs a{tables, table_stride, max_blocks, lens, held, free_blocks, free_capacity, free_count,
                new_tokens, num_requests, block_size, max_rows, rows, rows_stride, rows_width, slot_mapping,
                positions, cu_seqlens, kv_lens, refused, arrivals};
    if (int e = check_tables(a)) return e;
    if (!cu_seqlens || !refused || (num_requests > 0 && !kv_lens)) return MF_ERR_ARG;
    if (max_rows > 0 && (!slot_mapping || !positions)) return MF_ERR_ARG;
    if (rows && (rows_width < 0 || rows_stride < rows_width)) return MF_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    const int64_t shares = (max_rows + kThreads * kRowsPerThread - 1) / (kThreads * kRowsPerThread);
    if (rows && max_rows > 0) {
        const int64_t fill = std::min<int64_t>((max_rows + kThreads - 1) / kThreads, 1024);
        hipLaunchKernelGGL(fill_rows_kernel, dim3((unsigned)fill), dim3(kThreads), 0, st, slot_mapping, positions,
                           max_rows);
        if (int e = check_launch()) return e;
    }
    const int64_t by_rows = rows ? 1 : shares;
    const int64_t grid = std::min<int64_t>(std::max<int64_t>({by_rows, (int64_t)(num_requests + 3) / 4, 1}), 1024);
    hipLaunchKernelGGL(extend_kernel, dim3((unsigned)grid), dim3(kThreads), 0, st, a);
    return check_launch();
}

extern "C" int mf_tables_truncate(int32_t* tables, int64_t table_stride, int max_blocks, int32_t* lens, int32_t* held,
                                  int32_t* free_blocks, int64_t free_capacity, int32_t* free_count,
                                  const int32_t* lengths, int num_requests, int block_size, uint32_t* arrivals,
                                  mf_stream_t stream) {
    using namespace mf;
    TableArgs a{tables, table_stride, max_blocks, lens, held, free_blocks, free_capacity, free_count,
                lengths, num_requests, block_size, 0, nullptr, 0, 0, nullptr,
                nullptr, nullptr, nullptr, nullptr, arrivals};
    if (int e = check_tables(a)) return e;
    if (num_requests == 0) return MF_OK;
    const int grid = std::min((num_requests + 3) / 4, 1024);
    hipLaunchKernelGGL(truncate_kernel, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a);
    return check_launch();
}
