// The accepted path of a tree of drafted tokens.
//
// Node i of a sequence is drafted as a child of node parents[i] < i; node 0 is
// the sequence's newest token. A node is matched when its token is the one that
// the target drew from its parent's logits; of several matched siblings the
// first counts. The accepted path starts at node 0 and goes from each node to
// its matched child, so it emits the target's tokens at its nodes.
//
// One wave a sequence: every node offers itself to its parent (an LDS minimum
// per parent), then every lane follows the chain. Bound by latency: four dependent
// loads, and about 0.1 us for each accepted node (8 trees of 16 nodes 3.2 us on an
// MI355X, 256 of up to 64 3.6).
#include <algorithm>

#include "mf_common.h"

namespace mf {
namespace {

constexpr int kMaxNodes = MF_TREE_MAX_NODES;

struct AcceptArgs {
    const int64_t* tokens;
    const int64_t* targets;
    const int32_t* parents;
    const int32_t* cu_nodes;
    int num_seqs;
    int64_t num_rows;
    int max_nodes;
    int32_t* path;
    int64_t* out_tokens;
    int32_t* count;
};

__global__ __launch_bounds__(64) void accept_kernel(AcceptArgs a) {
    extern __shared__ int lds[];
    int* child = lds;                // each node's matched child, or max_nodes
    int* path = lds + a.max_nodes;
    const int s = blockIdx.x, lane = threadIdx.x;
    const int64_t first = a.cu_nodes[s], last = a.cu_nodes[s + 1];
    int n = (int)min(last - first, (int64_t)a.max_nodes);
    if (first < 0 || n < 0 || first + n > a.num_rows) n = 0;
    for (int i = lane; i < n; i += 64) child[i] = a.max_nodes;
    __syncthreads();
    for (int i = lane; i < n; i += 64) {
        const int p = a.parents[first + i];
        if (p >= 0 && p < i && a.tokens[first + i] == a.targets[first + p]) atomicMin(&child[p], i);
    }
    __syncthreads();
    int count = 0;
    if (n > 0) {  // the same walk in every lane; a child's number is above its parent's, so it ends
        for (int at = 0; at < n; at = child[at]) {
            if (lane == 0) path[count] = at;
            ++count;
        }
    }
    __syncthreads();
    for (int i = lane; i < a.max_nodes; i += 64) {
        const int64_t to = (int64_t)s * a.max_nodes + i;
        const int64_t row = i < count ? first + path[i] : -1;
        a.path[to] = (int)row;
        a.out_tokens[to] = row >= 0 ? a.targets[row] : -1;
    }
    if (lane == 0) a.count[s] = count;
}

}  // namespace
}  // namespace mf

extern "C" int mf_tree_accept(const int64_t* tokens, const int64_t* targets, const int32_t* parents,
                              const int32_t* cu_nodes, int num_seqs, int64_t num_rows, int max_nodes, int32_t* path,
                              int64_t* out_tokens, int32_t* count, mf_stream_t stream) {
    using namespace mf;
    if (num_seqs < 0 || num_rows < 0 || max_nodes < 1 || max_nodes > kMaxNodes) return MF_ERR_ARG;
    if (num_seqs == 0) return MF_OK;
    if (!cu_nodes || !path || !out_tokens || !count) return MF_ERR_ARG;
    if (num_rows > 0 && (!tokens || !targets || !parents)) return MF_ERR_ARG;
    AcceptArgs a{tokens, targets, parents, cu_nodes, num_seqs, num_rows, max_nodes, path, out_tokens, count};
    hipLaunchKernelGGL(accept_kernel, dim3((unsigned)num_seqs), dim3(64), 2 * max_nodes * sizeof(int),
                       (hipStream_t)stream, a);
    return check_launch();
}
