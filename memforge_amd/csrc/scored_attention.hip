// Attention whose scores are capped by a tanh, lowered by a bias that grows with
// the distance, or masked by documents and prefixes: the SC instances of the
// kernels in attn_kernels.h, in a file of their own so that they compile beside
// the plain ones.
//
// Per (row, key): t = scale * q.k; with a cap t = cap tanh(t / cap); with slopes
// t -= slope[head] |position - key|. Visible are the keys from the sequence's
// first one on that lie at or before the row's position, or inside the
// sequence's prefix. The rest is the plain kernels': the same tiles, plans,
// splits and merges, with the scores brought to log2 units before the running
// maximum instead of inside the exponent.
#include "attn_kernels.h"

namespace mf {

int launch_scored(int dtype, int dp, bool tail, const ScoredArgs& a, const int32_t* items, int64_t n_narrow,
                  int64_t n_wide, const int32_t* merges, int64_t n_merges, bool fast, const int32_t* dev_counts,
                  hipStream_t stream) {
#define MF_SCORED_CASE(DT, DPV)                                                                                     \
    if (dtype == DT && dp == DPV)                                                                                   \
        return tail ? launch_attention<DT, DPV, true, true>(a, items, n_narrow, n_wide, merges, n_merges, fast,     \
                                                            dev_counts, stream)                                     \
                    : launch_attention<DT, DPV, false, true>(a, items, n_narrow, n_wide, merges, n_merges, fast,    \
                                                             dev_counts, stream);
    MF_SCORED_CASE(MF_F32, 16)
    MF_SCORED_CASE(MF_F32, 32)
    MF_SCORED_CASE(MF_F32, 64)
    MF_SCORED_CASE(MF_F32, 128)
    MF_SCORED_CASE(MF_BF16, 32)
    MF_SCORED_CASE(MF_BF16, 64)
    MF_SCORED_CASE(MF_BF16, 128)
    MF_SCORED_CASE(MF_BF16, 256)
    MF_SCORED_CASE(MF_F16, 32)
    MF_SCORED_CASE(MF_F16, 64)
    MF_SCORED_CASE(MF_F16, 128)
    MF_SCORED_CASE(MF_F16, 256)
#undef MF_SCORED_CASE
    return MF_ERR_UNSUPPORTED;
}

}  // namespace mf
