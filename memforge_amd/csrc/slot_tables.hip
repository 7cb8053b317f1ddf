// Block tables and slot maps built on the device from request lengths: the
// growth of a batch by given numbers of tokens (blocks popped from a stack, a
// slot for every new token), and its cut back to given lengths (blocks pushed
// again).
//
// One launch each (growth with rows given by number: one more, which clears all
// rows first). Every workgroup scans the batch's lengths for itself (at most
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
constexpr int kWaveRows = 512;  // consecutive rows of one wave
constexpr int kWgRows = kWaveRows * kThreads / 64;

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
    int block_shift;      // -1: not a power of two
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
    if (gridDim.x == 1) return true;
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

__device__ __forceinline__ int block_of(const TableArgs& a, int pos) {
    return a.block_shift >= 0 ? pos >> a.block_shift : (int)((unsigned)pos / (unsigned)a.block_size);
}
__device__ __forceinline__ int64_t blocks_for(const TableArgs& a, int64_t tokens) {
    const int64_t up = tokens + a.block_size - 1;  // (lengths are below 2^32, so 32 bits hold all but refused ones)
    if (a.block_shift >= 0) return up >> a.block_shift;
    return up <= (int64_t)UINT_MAX ? (int64_t)((uint32_t)up / (uint32_t)a.block_size) : up / a.block_size;
}

// A request's state, clamped to what the tables hold, and what it asks for.
struct Request {
    int len, held, n;
};
__device__ __forceinline__ Request load_request(const TableArgs& a, int s) {
    return Request{max(a.lens[s], 0), min(max(a.held[s], 0), a.max_blocks), max(a.want[s], 0)};
}

// Measured (MI355X, kernel times): the slots of 847,366 rows of 256 requests 15.6 us, the cut
// back of their 53,000 blocks 9.8; of 106 rows of 8 requests 5.5 and 2.7. Latency at both: the
// lengths, the scan, then the blocks, then the stores (13.6 MB in the first, 2.8 us at a large
// copy's rate).
__global__ __launch_bounds__(kThreads) void extend_kernel(TableArgs a) {
    // the row each request starts at, the blocks taken before it (-1: it is refused), its state
    __shared__ int cu[kMaxRequests + 1], taken[kMaxRequests], lens[kMaxRequests], helds[kMaxRequests];
    const int B = a.num_requests, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = (B + kThreads - 1) / kThreads;
    const int s0 = min((int)threadIdx.x * per, B), s1 = min(s0 + per, B);
    const int count = (int)min(max((int64_t)*a.free_count, (int64_t)0), a.free_capacity);

    // ---- rows, then (of the requests that tables and rows suffice for) blocks
    int64_t rows = 0, total_rows;
    for (int s = s0; s < s1; ++s) {
        const Request r = load_request(a, s);
        lens[s] = r.len;
        helds[s] = r.held;
        cu[s] = r.n;
        rows += r.n;
    }
    int64_t row = block_scan(rows, total_rows);
    int64_t blocks = 0, total_blocks;
    for (int s = s0; s < s1; ++s) {
        const int n = cu[s];
        const int64_t need = blocks_for(a, (int64_t)lens[s] + n);
        cu[s] = clamp_count(row);
        row += n;
        const bool fits = need <= a.max_blocks && row <= a.max_rows && (int64_t)lens[s] + n <= INT_MAX &&
                          (a.rows == nullptr || n <= a.rows_width);
        taken[s] = fits ? (int)max(need - helds[s], (int64_t)0) : -1;  // for now: the blocks it lacks
        blocks += max(taken[s], 0);
    }
    if (threadIdx.x == kThreads - 1) cu[B] = clamp_count(total_rows);
    int64_t run = block_scan(blocks, total_blocks);
    int64_t refused = 0, all_refused, used = 0, total_used;
    for (int s = s0; s < s1; ++s) {
        const int grow = taken[s];
        run += max(grow, 0);
        const bool served = grow == 0 || (grow > 0 && run <= count);
        taken[s] = !served ? -1 : grow ? (int)(run - grow) : 0;
        refused += !served;
        used += served ? grow : 0;
    }
    block_scan(refused << 32 | used, all_refused);  // both below 2^31; with the scan's barriers, cu and taken are whole
    total_used = all_refused & 0xffffffff;
    all_refused >>= 32;
    __syncthreads();
    auto block_at = [&](int s, int j) -> int {
        const int held = helds[s];
        return j < held ? a.tables[(int64_t)s * a.table_stride + j] : a.free_blocks[count - 1 - (taken[s] + j - held)];
    };
    auto place = [&](int s, int pos, int64_t out) {
        const int j = block_of(a, pos);
        a.slot_mapping[out] = (int64_t)block_at(s, j) * a.block_size + (pos - j * a.block_size);
        a.positions[out] = pos;
    };

    // ---- this wave's share of the new tokens' rows
    if (a.rows == nullptr) {
        for (int64_t first = ((int64_t)blockIdx.x * (kThreads / 64) + wave) * kWaveRows; first < a.max_rows;
             first += (int64_t)gridDim.x * kWgRows) {
            int s = 0, hi = B - 1;  // the last request that starts at or before this lane's row
            while (s < hi) {
                const int mid = (s + hi + 1) >> 1;
                if (cu[mid] <= first + lane) s = mid;
                else hi = mid - 1;
            }
#pragma unroll 4
            for (int i = 0; i < kWaveRows / 64; ++i) {
                const int64_t r = first + 64 * i + lane;
                if (r >= a.max_rows) break;
                if (r < cu[B]) {
                    while (s + 1 < B && cu[s + 1] <= r) ++s;
                    const int64_t pos = (int64_t)lens[s] + (r - cu[s]);
                    if (taken[s] >= 0) {
                        place(s, (int)pos, r);
                    } else {
                        a.slot_mapping[r] = -1;
                        a.positions[r] = pos;
                    }
                } else {
                    a.slot_mapping[r] = -1;
                    a.positions[r] = 0;
                }
            }
        }
    }

    // ---- its share of the requests: fresh table entries, and rows given by number
    for (int s = (int)blockIdx.x * (kThreads / 64) + wave; s < B; s += (int)gridDim.x * (kThreads / 64)) {
        if (taken[s] < 0) continue;
        const int n = cu[s + 1] - cu[s], held = helds[s];
        const int grow = (int)max(blocks_for(a, (int64_t)lens[s] + n) - held, (int64_t)0);
        int32_t* trow = a.tables + (int64_t)s * a.table_stride;
        for (int j = lane; j < grow; j += 64) trow[held + j] = a.free_blocks[count - 1 - (taken[s] + j)];
        if (a.rows != nullptr) {
            for (int j = lane; j < n; j += 64) {
                const int out = a.rows[(int64_t)s * a.rows_stride + j];
                if (out >= 0 && out < a.max_rows) place(s, lens[s] + j, out);
            }
        }
    }
    if (blockIdx.x == 0) {
        for (int s = (int)threadIdx.x; s <= B; s += kThreads) a.cu_seqlens[s] = cu[s];
        if (threadIdx.x == 0) *a.refused = (int)all_refused;
    }

    // ---- the new state
    if (!last_to_finish(a.arrivals)) return;
    for (int s = (int)threadIdx.x; s < B; s += kThreads) {
        const bool served = taken[s] >= 0;
        const int len = lens[s] + (served ? cu[s + 1] - cu[s] : 0);
        a.lens[s] = len;
        a.kv_lens[s] = len;
        a.held[s] = served ? max(helds[s], (int)blocks_for(a, len)) : helds[s];
    }
    if (threadIdx.x == 0) *a.free_count = count - (int)total_used;
}

__global__ __launch_bounds__(kThreads) void truncate_kernel(TableArgs a) {
    __shared__ int before[kMaxRequests], kept[kMaxRequests], helds[kMaxRequests];  // before: blocks that earlier ones return
    const int B = a.num_requests, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int per = (B + kThreads - 1) / kThreads;
    const int s0 = min((int)threadIdx.x * per, B), s1 = min(s0 + per, B);
    const int64_t count = min(max((int64_t)*a.free_count, (int64_t)0), a.free_capacity);
    int64_t back = 0, total;
    for (int s = s0; s < s1; ++s) {
        const Request r = load_request(a, s);
        kept[s] = (int)min(blocks_for(a, min(r.n, r.len)), (int64_t)r.held);
        helds[s] = r.held;
        back += r.held - kept[s];
    }
    int64_t run = block_scan(back, total);
    for (int s = s0; s < s1; ++s) {
        before[s] = (int)run;
        run += helds[s] - kept[s];
    }
    __syncthreads();
    // the last block taken by the last request that grew lies on top again
    for (int s = (int)blockIdx.x * (kThreads / 64) + wave; s < B; s += (int)gridDim.x * (kThreads / 64)) {
        const int keep = kept[s], held = helds[s];
        int32_t* trow = a.tables + (int64_t)s * a.table_stride;
        for (int j = keep + lane; j < held; j += 64) {
            const int64_t place = count + total - 1 - (before[s] + j - keep);
            if (place < a.free_capacity) a.free_blocks[place] = trow[j];
            trow[j] = 0;
        }
    }
    if (!last_to_finish(a.arrivals)) return;
    for (int s = (int)threadIdx.x; s < B; s += kThreads) {
        const int len = max(a.lens[s], 0);
        a.lens[s] = min(len, max(a.want[s], 0));
        a.held[s] = kept[s];
    }
    if (threadIdx.x == 0) *a.free_count = (int)min(count + total, a.free_capacity);
}

int shift_of(int block_size) {
    for (int b = 0; b < 31; ++b)
        if (1 << b == block_size) return b;
    return -1;
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
                new_tokens, num_requests, block_size, shift_of(block_size), max_rows, rows, rows_stride, rows_width, slot_mapping,
                positions, cu_seqlens, kv_lens, refused, arrivals};
    if (int e = check_tables(a)) return e;
    if (!cu_seqlens || !refused || (num_requests > 0 && !kv_lens)) return MF_ERR_ARG;
    if (max_rows > 0 && (!slot_mapping || !positions)) return MF_ERR_ARG;
    if (rows && (rows_width < 0 || rows_stride < rows_width)) return MF_ERR_ARG;
    hipStream_t st = (hipStream_t)stream;
    const int64_t shares = (max_rows + kWgRows - 1) / kWgRows;
    if (rows && max_rows > 0) {
        const int64_t fill = std::min<int64_t>((max_rows + kThreads - 1) / kThreads, 1024);
        hipLaunchKernelGGL(fill_rows_kernel, dim3((unsigned)fill), dim3(kThreads), 0, st, slot_mapping, positions,
                           max_rows);
        if (int e = check_launch()) return e;
    }
    const int64_t by_rows = rows ? 1 : shares;
    const int64_t grid = std::min<int64_t>(std::max<int64_t>({by_rows, (int64_t)(num_requests + 15) / 16, 1}), 1024);
    hipLaunchKernelGGL(extend_kernel, dim3((unsigned)grid), dim3(kThreads), 0, st, a);
    return check_launch();
}

extern "C" int mf_tables_truncate(int32_t* tables, int64_t table_stride, int max_blocks, int32_t* lens, int32_t* held,
                                  int32_t* free_blocks, int64_t free_capacity, int32_t* free_count,
                                  const int32_t* lengths, int num_requests, int block_size, uint32_t* arrivals,
                                  mf_stream_t stream) {
    using namespace mf;
    TableArgs a{tables, table_stride, max_blocks, lens, held, free_blocks, free_capacity, free_count,
                lengths, num_requests, block_size, shift_of(block_size), 0, nullptr, 0, 0, nullptr,
                nullptr, nullptr, nullptr, nullptr, arrivals};
    if (int e = check_tables(a)) return e;
    if (num_requests == 0) return MF_OK;
    const int grid = (num_requests + 15) / 16;
    hipLaunchKernelGGL(truncate_kernel, dim3((unsigned)grid), dim3(kThreads), 0, (hipStream_t)stream, a);
    return check_launch();
}
