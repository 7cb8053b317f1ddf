// One token per row of logits from a given uniform number: temperature, top-k,
// top-p and min-p, then a draw by rank.
//
// A row's tokens are ranked by (logit descending, index ascending) and weighted by
// w = exp((logit - largest) / T). Every filter keeps a prefix of that ranking:
// top-k its first k, top-p the tokens with at most p of the first k's mass before
// them, min-p those of at least p of the largest weight. The drawn token is the
// first whose inclusive mass exceeds u times the kept mass. So all of it is
// positions in one running sum, and no sort is needed: the row is binned by
// logit, finely (256 bins to a factor e of weight), the bins in which a boundary
// lies are found from the bins' counts and masses, and only those bins' tokens
// are ranked.
//
// Exactness. A boundary between two tokens must fall where 64-bit arithmetic puts
// it, in sums over a whole vocabulary. A bin's mass is T_b (n - sum q) with T_b the
// weight at the bin's top, n its count and q = 1 - w / T_b < 2^-8. The q are formed
// in fp64 by a polynomial (error 2^-47) and added as integers, count and sum in one
// 64-bit LDS add, so the sums do not depend on their order. One is rounded to
// 2^-QS, QS = 71 - 2 log2(vocabulary), at most 40: 2^-37 at 131,072 tokens.
// Weights below e^-32 of the largest logit seen first (1e-14) count as nothing.
//
// Bins reach from 28 factors e above the largest logit of the row's first piece to
// 32 below it, so one pass serves what follows; a row with a logit above that
// range is binned again from its true maximum.
//
// Measured (MI355X, graph replays, us a call; floor: the logits read once at the 4.9 TB/s of a large copy):
// 256 rows of 130,021 fp32 logits, top_p 0.95: 80 (floor 27); 272 rows of 49,152 fp32: 60 (11;
// sixteen rows more than compute units); 64 rows of bf16, settings of every kind: 39; one row:
// 32. Of the 80: binning 43 (its loads alone 30, so memory before its 11 fp64 operations a token),
// the second pass, which looks for the boundary bins' tokens, 23, searches 4, ranking 9. Counters:
// the L2 fetches 271 MB, so both passes read the 133 MB of rows from behind it (64 rows of 49,152 in
// bf16: 6.9 of 6.3, once); vector instructions take 36 us of every SIMD (22.3 M), conflicts in
// LDS 8 us. A version with whole bins walked by single threads took 142.
//
// Slow by nature: a row whose peak lies more than 28 T above its first 8,192 logits is binned twice,
// and a split row is then taken whole (one row of 130,021: 79 us for 36 to 50; of 49,152 53 for 40; 256
// rows of 130,021: 78 for 58 to 65). Rows of equal logits, whose adds meet in one bin and whose boundaries are found by
// descent: 0.6 ms (no filter) to 1.1 (three) a call for one row or 64 of 49,152, 1.3 to 2.6 for one
// or 256 of 130,021.
#include <algorithm>

#include "mf_common.h"

namespace mf {
namespace {

constexpr int kThreads = 1024;
constexpr int kOwn = 15;                 // consecutive bins of one thread (odd: no LDS bank twice)
constexpr int kBins = kOwn * kThreads;
constexpr double kPerE = 256.0;          // bins to a factor e of weight
// The bin of the reference logit: 32 factors e below it have bins. Even and its thread's first,
// so that equal logits at the reference weigh exactly 1 (Binner, Owner).
constexpr int kTop = (kBins - 32 * 256) / (2 * kOwn) * (2 * kOwn);
static_assert(kTop % 2 == 0 && kTop % kOwn == 0 && kBins - kTop >= 8192, "the reference's bin");
constexpr int kList = 2048;              // tokens of boundary bins that are ranked in LDS
constexpr int kSegs = 128;               // boundary bins
constexpr int kFirst = 8192;             // tokens of a row whose maximum is the reference
constexpr int kRowWords = kBins + 2;     // a split row's bins, its largest (key, index), and its reference

struct SampleArgs {
    const char* logits;
    int64_t stride_row;
    int vocab;
    int num_rows;
    const float* uniforms;
    const float* temp;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    float temp0, top_p0, min_p0;
    int top_k0;
    int count_shift;  // a bin's word: count << count_shift | sum of q * 2^qs
    double q_scale, q_unit;  // 2^qs, 2^-qs
    int64_t* tokens;
    float* probs;
    uint64_t* bins;  // rows split over workgroups: kRowWords words a row, all 0 between calls
    int chunk;       // tokens of one workgroup's part
};

struct Seg {
    double mass_before;  // of the bins before it
    double top;          // T_b
    uint64_t total;      // sum of its tokens' 2^qs (1 - q)
    int bin, base, n, count_before, cursor;
};

// A bin that a search found (bin < 0: none).
struct Found {
    int bin, n, count_before;
    double mass_before, mass;
};

// Places of the searches' results.
enum { AT_K, AT_FIRST, AT_P_LO, AT_P_HI, AT_M, AT_D_LO, AT_D_HI, kFinds };

struct Shared {
    uint64_t words[kBins + 64];  // the bins, and words that are never read; then the ranking's arrays
    uint64_t list[kList];
    uint8_t list_seg[kList];
    Seg seg[kSegs];
    double wave_mass[16];
    int wave_count[16];
    float wave_max[16];
    unsigned long long best;
    int found[2];
    Found at[kFinds];
    int segs, listed;
    double d0, d1;
    uint64_t u0;
    int i0;
};

template <int DT>
__device__ __forceinline__ float value_of(uint32_t bits) {
    return bits_to_f32<DT>(bits);
}

// g(first index, 16 bytes of consecutive logits) for the tokens [e0, e1) of a row, each by one
// of the workgroup's threads, from the first aligned token on; f(index, logit) for the few
// around them.
template <int DT, class F, class G>
__device__ __forceinline__ void scan_row(const char* row, int e0, int e1, F f, G g) {
    constexpr int ES = DT == MF_F32 ? 4 : 2, VE = 16 / ES;
    const int tid = threadIdx.x;
    auto one = [&](int i) {
        f(i, value_of<DT>(ES == 4 ? ((const uint32_t*)row)[i] : (uint32_t)((const uint16_t*)row)[i]));
    };
    const int head = min((int)((16 - ((uintptr_t)(row + (int64_t)e0 * ES) & 15)) & 15) / ES, e1 - e0);
    if (tid < head) one(e0 + tid);
    const int v0 = e0 + head, nv = (e1 - v0) / VE;
    const uint4* vec = (const uint4*)(row + (int64_t)v0 * ES);
    // loads two rounds of U ahead, none of them behind a branch (the compiler waits for every
    // load in flight where a branch joins); past the end the last piece is read again
    constexpr int U = 2;
    if (nv > 0) {
        auto piece = [&](int w) { return vec[min(w, nv - 1)]; };
        uint4 one_ahead[U], two_ahead[U];
#pragma unroll
        for (int u = 0; u < U; ++u) one_ahead[u] = piece(tid + u * kThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) two_ahead[u] = piece(tid + (U + u) * kThreads);
        for (int v = tid; v < nv; v += U * kThreads) {
            uint4 cur[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                cur[u] = one_ahead[u];
                one_ahead[u] = two_ahead[u];
                two_ahead[u] = piece(v + (2 * U + u) * kThreads);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t x[4] = {cur[u].x, cur[u].y, cur[u].z, cur[u].w};
                float v_[VE];
#pragma unroll
                for (int k = 0; k < VE; ++k)
                    v_[k] = value_of<DT>(ES == 4 ? x[k] : (k & 1 ? x[k >> 1] >> 16 : x[k >> 1] & 0xffffu));
                if (v + u * kThreads < nv) g(v0 + (v + u * kThreads) * VE, v_);
            }
        }
    }
    const int tail = v0 + nv * VE;
    if (tid < e1 - tail) one(tail + tid);
}
template <int DT, class F>
__device__ __forceinline__ void scan_row(const char* row, int e0, int e1, F f) {
    scan_row<DT>(row, e0, e1, f, [&](int i, const auto& v) {
#pragma unroll
        for (int k = 0; k < (int)(sizeof(v) / 4); ++k) f(i + k, v[k]);
    });
}

// Larger for a larger logit; -0 as 0, NaN as -infinity.
__device__ __forceinline__ uint32_t order_key(float v) {
    const uint32_t u = v == v ? __float_as_uint(v + 0.f) : 0xff800000u;
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

// Places of logits below a finite reference: y = kTop + 256 (reference - logit) / T, whose whole
// part is the bin: y - 1/2 rounded to the nearest, which leaves the whole number in the low
// bits of a sum and costs a quarter of the conversions (a y that is whole may fall to the
// bin above, with the same weight; the even kTop itself does not).
struct Binner {
    double ref, per, c1, c2, c3, c4;
    uint32_t one_hi;  // a token's count in its word
    float lo, hi;     // the logits that have a bin

    static constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52
    __device__ __forceinline__ Binner(const SampleArgs& a, float reference, float temp)
        : ref(reference), per(kPerE / (double)temp), c1(a.q_scale), c2(-0.5 * a.q_scale), c3(a.q_scale / 6.0),
          c4(a.q_scale / -24.0), one_hi(1u << (a.count_shift - 32)) {
        lo = fmaxf((float)(ref - (kBins - kTop - 0.02) / per), -3.4028234663852886e38f);
        hi = fminf((float)(ref + (kTop - 0.02) / per), 3.4028234663852886e38f);
        while (!(y_of(lo) < kBins - 0.01)) lo = nextafterf(lo, __builtin_huge_valf());  // rounded outwards: a step or two
        while (!(y_of(hi) > 0.01)) hi = nextafterf(hi, -__builtin_huge_valf());
    }
    __device__ __forceinline__ double y_of(float v) const { return __builtin_fma(ref - (double)v, per, (double)kTop); }
    // a token's bin and its place below the bin's top in factors e; false where it has none
    __device__ __forceinline__ bool has_bin(float v) const { return v >= lo && v <= hi; }
    __device__ __forceinline__ void place_any(float v, int& bin, double& t) const {
        const double y = __builtin_fma(ref - (double)v, per, kTop - 0.5), whole = y + kWhole;
        bin = (int)(uint32_t)__double_as_longlong(whole);
        t = __builtin_fma(y - (whole - kWhole), 1.0 / kPerE, 0.5 / kPerE);
    }
    __device__ __forceinline__ bool place(float v, int& bin, double& t) const {
        if (!has_bin(v)) return false;
        place_any(v, bin, t);
        return true;
    }
    // 2^qs q, q = 1 - exp(-t)
    __device__ __forceinline__ uint32_t q_of(double t) const {
        return (uint32_t)__double_as_longlong(
            __builtin_fma(t, __builtin_fma(t, __builtin_fma(t, __builtin_fma(t, c4, c3), c2), c1), 4503599627370496.0));
    }
    __device__ __forceinline__ unsigned long long word(double t) const { return (unsigned long long)one_hi << 32 | q_of(t); }
    // a number below every logit of bins up to `bin`
    __device__ __forceinline__ float value_below(int bin) const {
        const double v = ref - ((double)(bin - kTop) + 1.1) / per;
        return (float)(v - fabs(v) * 1e-6);
    }
};

__device__ __forceinline__ double bin_top(int bin) { return exp((double)(kTop - bin) * (1.0 / kPerE)); }

__device__ __forceinline__ float block_max(Shared& sh, float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave_max[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = sh.wave_max[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) m = fmaxf(m, sh.wave_max[w]);
    return m;
}

__device__ __forceinline__ void clear_words(Shared& sh) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.words[i] = 0;
}

// Exclusive sums of the threads' counts and masses, and the totals; mass_end: the inclusive
// sum, to the bit the next thread's exclusive one.
__device__ __forceinline__ void block_sums(Shared& sh, int& n, double& mass, double& mass_end, int& n_all, double& mass_all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int ni = n;
    double mi = mass;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int nu = __shfl_up(ni, o, 64);
        const double mu = __shfl_up(mi, o, 64);
        if (lane >= o) {
            ni += nu;
            mi += mu;
        }
    }
    double before = __shfl_up(mi, 1, 64);
    if (lane == 0) before = 0.0;
    __syncthreads();
    if (lane == 63) {
        sh.wave_count[wave] = ni;
        sh.wave_mass[wave] = mi;
    }
    __syncthreads();
    int nb = 0;
    double mb = 0.0;
    n_all = 0;
    mass_all = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w == wave) {
            nb = n_all;
            mb = mass_all;
        }
        n_all += sh.wave_count[w];
        mass_all += sh.wave_mass[w];
    }
    n = nb + ni - n;
    mass = mb + before;
    mass_end = mb + mi;
}

// The bins of one thread.
struct Owner {
    int count_shift;
    double q_scale, q_unit;
    int count_before, count_end;      // of the bins before this thread's, and with them
    double mass_before, mass_end;
    double top0;                      // T_b of its first bin
    double down;                      // exp(-lane / 256)

    // from the bins in sh.words, with the totals; empties the searches' places
    __device__ __forceinline__ void build(const SampleArgs& a, Shared& sh, int& n_all, double& mass_all) {
        count_shift = a.count_shift;
        q_scale = a.q_scale;
        q_unit = a.q_unit;
        count_before = 0;
        mass_before = 0.0;
        top0 = bin_top(threadIdx.x * kOwn);
        down = exp((double)(threadIdx.x & 63) * (-1.0 / kPerE));
        int n = 0;
        double mass = 0.0;
        walk(sh, [&](int, uint64_t w, double, int, double, double m) {
            n += count(w);
            mass += m;
        });
        if (threadIdx.x < kFinds) sh.at[threadIdx.x].bin = -1;
        int before = n;
        block_sums(sh, before, mass, mass_end, n_all, mass_all);
        count_before = before;
        mass_before = mass;
        count_end = before + n;
    }

    __device__ __forceinline__ static double step() { return 0.9961013694701175; }  // exp(-1/256)
    __device__ __forceinline__ int count(uint64_t w) const { return (int)(w >> count_shift); }
    __device__ __forceinline__ uint64_t parts(uint64_t w) const {
        const uint64_t n = w >> count_shift;
        return n * (uint64_t)q_scale - (w & ((1ull << count_shift) - 1));
    }
    // n - sum of q: the word's weight in units of T_b (its sum is below 2^52)
    __device__ __forceinline__ double weight(uint64_t w) const {
        const double q = __longlong_as_double((long long)((w & ((1ull << count_shift) - 1)) | 0x4330000000000000ull)) - 4503599627370496.0;
        return __builtin_fma(q, -q_unit, (double)(uint32_t)(w >> count_shift));
    }
    // g(bin, word, T_b, count before, mass before, mass) for every bin that holds anything
    template <class G>
    __device__ __forceinline__ void walk(const Shared& sh, G g) const {
        double top = top0, before = mass_before;
        int n = count_before;
#pragma unroll 5
        for (int j = 0; j < kOwn; ++j) {
            const uint64_t w = sh.words[threadIdx.x * kOwn + j];
            if (w) {
                const double mass = top * weight(w);
                g((int)threadIdx.x * kOwn + j, w, top, n, before, mass);
                before += mass;
                n += count(w);
            }
            top *= step();
        }
    }
};

__device__ __forceinline__ double top_of(int bin) {  // T_b as its owner forms it
    double t = bin_top(bin / kOwn * kOwn);
    for (int j = 0; j < bin % kOwn; ++j) t *= Owner::step();
    return t;
}

// The first bin whose inclusive mass exceeds x (COUNT: whose inclusive count does), into
// sh.at[k], which holds bin -1 before and where there is none. One thread's bins hold the
// crossing, so nothing is compared between threads; the caller's next barrier publishes it.
// The owner's wave works out its bins side by side.
template <bool COUNT>
__device__ __forceinline__ void find(Shared& sh, const Owner& o, double x, int k) {
    const uint64_t owner = __builtin_amdgcn_ballot_w64(
        COUNT ? (double)o.count_before <= x && (double)o.count_end > x : o.mass_before <= x && o.mass_end > x);
    if (owner == 0) return;
    const int src = __ffsll((unsigned long long)owner) - 1, lane = threadIdx.x & 63;
    const double base = __shfl(o.mass_before, src, 64);
    const int base_n = __shfl(o.count_before, src, 64);
    const int bin = ((int)threadIdx.x - lane + src) * kOwn + lane;
    const uint64_t w = lane < kOwn ? sh.words[bin] : 0;
    const double top = __shfl(o.top0, src, 64) * o.down;
    const double mass = w ? top * o.weight(w) : 0.0;
    const int n = o.count(w);
    double upto = mass;
    int upto_n = n;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        const double m1 = __shfl_up(upto, d, 64);
        const int n1 = __shfl_up(upto_n, d, 64);
        if (lane >= d) {
            upto += m1;
            upto_n += n1;
        }
    }
    const uint64_t held = __builtin_amdgcn_ballot_w64(w != 0);
    const uint64_t past = __builtin_amdgcn_ballot_w64(w != 0 && (COUNT ? (double)(base_n + upto_n) > x : base + upto > x));
    // (these sums round differently from the owner's: without a crossing the last bin stands in)
    const int at = past ? __ffsll((unsigned long long)past) - 1 : 63 - __clzll((long long)held);
    if (lane == at) sh.at[k] = Found{bin, n, base_n + upto_n - n, base + upto - mass, mass};
}

// A prefix of the ranking: whole bins before `bin`, then the first n tokens of it.
struct Limit {
    int bin, n;
    double mass;  // of the prefix
    __device__ __forceinline__ bool before(const Limit& o) const { return bin < o.bin || (bin == o.bin && n < o.n); }
};

// Boundary bins too full for the list: the token at which a running sum over the
// bin's ranking passes a target is found digit by digit, from 64-bit rank keys
// (logit key inverted, then index) of which every level bins the next 12 bits. Six
// passes over the row; rows of many equal logits and extreme temperatures.
struct Ranked {
    uint64_t key;          // of the token found
    int before;            // tokens of the bin ranked before it
    double parts_before;   // and their sum of 2^qs (1 - q)
    double parts;          // its own
    bool found;
};

__device__ __forceinline__ uint64_t parts_in(const SampleArgs& a, uint64_t w) {
    return (w >> a.count_shift) * (uint64_t)a.q_scale - (w & ((1ull << a.count_shift) - 1));
}

template <int DT>
__device__ __forceinline__ Ranked descend(const SampleArgs& a, Shared& sh, const char* row, const Binner& bn, int bin, bool by_count,
                          double target) {
    // target: tokens (by_count) or parts; found is the first whose inclusive sum exceeds it
    Ranked r{0, 0, 0.0, 0.0, true};
    uint64_t prefix = 0;
    for (int level = 0; level < 6; ++level) {
        const int shift = level < 5 ? 52 - 12 * level : 0;
        const int width = level < 5 ? 12 : 4;
        __syncthreads();
        for (int i = threadIdx.x; i < 4096; i += kThreads) sh.words[i] = 0;
        __syncthreads();
        scan_row<DT>(row, 0, a.vocab, [&](int i, float v) {
            int at;
            double part;
            if (!bn.place(v, at, part) || at != bin) return;
            const uint64_t key = (uint64_t)~order_key(v) << 32 | (uint32_t)i;
            if (level > 0 && (key >> (shift + width)) != prefix) return;
            atomicAdd((unsigned long long*)&sh.words[(key >> shift) & ((1u << width) - 1)],
                      bn.word(part));
        });
        __syncthreads();
        // four digits to a thread: the first whose inclusive sum passes the target, else the last
        int n = 0, n_before, n_all;
        double parts = 0.0, parts_before, parts_end, parts_all;
        uint64_t w[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            w[d] = sh.words[4 * threadIdx.x + d];
            n += (int)(w[d] >> a.count_shift);
            parts += (double)parts_in(a, w[d]);
        }
        n_before = n;
        parts_before = parts;
        block_sums(sh, n_before, parts_before, parts_end, n_all, parts_all);
        if (threadIdx.x == 0) {
            sh.found[0] = 4096;
            sh.found[1] = -1;
        }
        __syncthreads();
        n_before += r.before;
        parts_before += r.parts_before;
        int pick = 4096, last = -1, at_n = 0;
        double at_parts = 0.0, own = 0.0, last_parts = 0.0, last_own = 0.0;
        int last_n = 0;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            if (!w[d]) continue;
            const int dn = (int)(w[d] >> a.count_shift);
            const double dp = (double)parts_in(a, w[d]);
            last = 4 * threadIdx.x + d;
            last_n = n_before;
            last_parts = parts_before;
            last_own = dp;
            if (pick == 4096 && (by_count ? (double)(n_before + dn) > target : parts_before + dp > target)) {
                pick = last;
                at_n = n_before;
                at_parts = parts_before;
                own = dp;
            }
            n_before += dn;
            parts_before += dp;
        }
        if (pick < 4096) atomicMin(&sh.found[0], pick);
        if (last >= 0) atomicMax(&sh.found[1], last);
        __syncthreads();
        const bool passed = sh.found[0] < 4096;
        if (sh.found[1] < 0 || (level == 0 && !passed)) {
            r.found = false;
            return r;
        }
        const int digit = passed ? sh.found[0] : sh.found[1];
        if (passed ? pick == digit : last == digit) {
            sh.i0 = passed ? at_n : last_n;
            sh.d0 = passed ? at_parts : last_parts;
            sh.d1 = passed ? own : last_own;
        }
        __syncthreads();
        prefix = prefix << width | (uint64_t)digit;
        r.before = sh.i0;
        r.parts_before = sh.d0;
        r.parts = sh.d1;
    }
    r.key = prefix;
    return r;
}

// Bins of the tokens [e0, e1) into sh.words; their largest logit.
template <int DT>
__device__ float bin_range(const SampleArgs& a, Shared& sh, const char* row, const Binner& bn, int e0, int e1) {
    float m = -__builtin_huge_valf();
    auto add = [&](int bin, double part) { atomicAdd((unsigned long long*)&sh.words[bin], bn.word(part)); };
    scan_row<DT>(
        row, e0, e1,
        [&](int, float v) {
            m = fmaxf(m, v);
            int bin;
            double part;
            if (bn.place(v, bin, part)) add(bin, part);
        },
        [&](int, const auto& v) {
            // without a branch between them, so that their chains of fp64 operations run side by
            // side; what has no bin adds to a word of the lane's own
            constexpr int N = sizeof(v) / 4;
            int bin[N];
            unsigned long long word[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                m = fmaxf(m, v[k]);
                double part;
                bn.place_any(v[k], bin[k], part);
                bin[k] = bn.has_bin(v[k]) ? bin[k] : kBins + (int)(threadIdx.x & 63);
                word[k] = bn.word(part);
            }
#pragma unroll
            for (int k = 0; k < N; ++k) atomicAdd((unsigned long long*)&sh.words[bin[k]], word[k]);
        });
    return block_max(sh, m);
}

// The finish of a row whose boundary bins are too full for the list: each boundary by itself,
// in the same order (see descend). Rows of many equal logits and extreme temperatures.
// top_k 0, p_of -1, mb kBins: no such filter; sh.at holds the searches for k, m and the first.
template <int DT>
__device__ __forceinline__ void finish_full(const SampleArgs& a, Shared& sh, const char* row, int r, const Binner& bn, double u,
                                            int top_k, double p_of, double least, int mb, double mass_all) {
    const int tid = threadIdx.x;
    const Found at_k = sh.at[AT_K], at_m = sh.at[AT_M];
    const int first_bin = sh.at[AT_FIRST].bin;
    Limit limit{kBins, 0, mass_all};
    if (mb != kBins) {
        const double top = top_of(mb);
        __syncthreads();
        if (tid == 0) {
            sh.u0 = 0;
            sh.i0 = 0;
        }
        __syncthreads();
        scan_row<DT>(row, 0, a.vocab, [&](int, float v) {
            int at;
            double part;
            if (!bn.place(v, at, part) || at != mb) return;
            const uint64_t p = (uint64_t)a.q_scale - bn.q_of(part);
            if (top * ((double)p * a.q_unit) < least) return;
            atomicAdd((unsigned long long*)&sh.u0, (unsigned long long)p);
            atomicAdd(&sh.i0, 1);
        });
        __syncthreads();
        limit = Limit{mb, sh.i0, at_m.mass_before + top * ((double)sh.u0 * a.q_unit)};
    }
    double mass_k = mass_all;
    enum { BY_K, BY_P, ONE, DRAW, LAST };
    bool clobbered = false;  // a descent has used the bins' memory
    for (int stage = BY_K; stage <= LAST; ++stage) {
        // ---- the bin, and the count or mass whose passing is looked for
        Found f{-1, 0, 0, 0.0, 0.0};
        bool by_count = false;
        double target = 0.0;
        if (stage == BY_K) {
            if (top_k == 0) continue;
            f = at_k;
            by_count = true;
            target = (double)(top_k - 1 - f.count_before);
        } else if (stage == ONE) {
            f.bin = first_bin;
            by_count = true;
        } else {
            if (stage == BY_P && p_of < 0.0) continue;
            if (stage != LAST) {
                const double x = stage == BY_P ? p_of * mass_k : u * limit.mass;
                __syncthreads();
                if (clobbered) {
                    clear_words(sh);
                    __syncthreads();
                    bin_range<DT>(a, sh, row, bn, 0, a.vocab);
                    __syncthreads();
                }
                Owner own;
                int n_all;
                double m_all;
                own.build(a, sh, n_all, m_all);
                __syncthreads();
                find<false>(sh, own, x, AT_D_LO);
                __syncthreads();
                f = sh.at[AT_D_LO];
                target = (x - f.mass_before) / top_of(max(f.bin, 0)) * a.q_scale;
                if (stage == BY_P && f.bin < 0) continue;
                if (stage == DRAW && (f.bin < 0 || f.bin > limit.bin)) continue;  // the limit's last token
            } else {
                f.bin = limit.bin;
                by_count = true;
                target = (double)(limit.n - 1);
            }
        }
        const double top = top_of(f.bin);
        const Ranked e = descend<DT>(a, sh, row, bn, f.bin, by_count, target);
        clobbered = true;
        const double upto = f.mass_before + top * ((e.parts_before + e.parts) * a.q_unit);
        if (stage == BY_K) {
            const Limit l{f.bin, e.before + 1, upto};
            mass_k = l.mass;
            if (l.before(limit)) limit = l;
        } else if (stage == BY_P) {
            const Limit l = e.found ? Limit{f.bin, e.before + 1, upto} : Limit{f.bin, f.n, f.mass_before + f.mass};
            if (l.before(limit)) limit = l;
        } else if (stage == ONE) {
            const Limit l{f.bin, 1, top * (e.parts * a.q_unit)};
            if (limit.before(l)) limit = l;
        } else {
            if (stage == DRAW) {
                if (!e.found && f.bin != limit.bin) {  // the bin's last token, by a rounding
                    limit = Limit{f.bin, f.n, limit.mass};
                    continue;
                }
                if (!e.found || (f.bin == limit.bin && e.before >= limit.n)) continue;
            }
            if (tid == 0) {
                a.tokens[r] = (int64_t)(uint32_t)e.key;
                if (a.probs) a.probs[r] = (float)(top * (e.parts * a.q_unit) / limit.mass);
            }
            __syncthreads();
            return;
        }
    }
}

// The finish of one row, whose bins are in sh.words.
template <int DT, bool FULL>
__device__ __forceinline__ void finish_row(const SampleArgs& a, Shared& sh, const char* row, int r, const Binner& bn, float largest) {
    const int tid = threadIdx.x;
    Owner own;
    int n_all;
    double mass_all;
    own.build(a, sh, n_all, mass_all);

    const int top_k = a.top_k ? a.top_k[r] : a.top_k0;
    const double top_p = a.top_p ? a.top_p[r] : a.top_p0;
    const double min_p = a.min_p ? a.min_p[r] : a.min_p0;
    double u = a.uniforms[r];
    u = u > 0.0 ? fmin(u, 1.0 - 0x1p-24) : 0.0;

    // ---- the bins in which the boundaries lie. Exact masses need a bin's tokens:
    // until then a boundary is an interval of bins.
    const bool by_k = top_k > 0 && top_k < n_all;
    const bool by_p = !(top_p >= 1.0);
    const bool by_m = min_p > 0.0;
    const int none = kBins;
    // the least weight that min_p lets pass, in the bins' unit
    // (formed as the tokens' own weights are, so that one passes at 1)
    int top_bin = 0;
    double top_part = 0.0;
    bn.place(largest, top_bin, top_part);
    const double least = min_p * (top_of(top_bin) * ((double)((uint64_t)a.q_scale - bn.q_of(top_part)) * a.q_unit));
    int kb = none, p_lo = none, p_hi = none, mb = none;
    double lo = mass_all, hi = mass_all;
    if (by_k) find<true>(sh, own, (double)(top_k - 1), AT_K);
    find<true>(sh, own, 0.0, AT_FIRST);  // the first bin that holds anything
    if (by_m) {
        // w >= min_p: places down to -ln(min_p) below the largest logit
        const double y = bn.y_of(largest), edge = min_p > 1.0 ? y : y - log(min_p) * kPerE;
        mb = edge < kBins - 1 ? max((int)floor(edge), 0) : none;
        if (mb != none && tid == mb / kOwn) {  // the masses around that bin
            double before = own.mass_before, m = 0.0;
            own.walk(sh, [&](int bin, uint64_t, double, int, double b, double mm) {
                if (bin < mb) before = b + mm;
                if (bin == mb) m = mm;
            });
            sh.at[AT_M] = Found{mb, 0, 0, before, m};
        }
    }
    __syncthreads();
    const int first_bin = sh.at[AT_FIRST].bin;
    if (by_k) {
        kb = sh.at[AT_K].bin;
        lo = sh.at[AT_K].mass_before;
        hi = lo + sh.at[AT_K].mass;
    }
    const double p_of = top_p > 0.0 ? top_p : 0.0;
    if (by_p) {
        find<false>(sh, own, p_of * lo, AT_P_LO);
        find<false>(sh, own, p_of * hi, AT_P_HI);
        __syncthreads();
        p_lo = sh.at[AT_P_LO].bin >= 0 ? sh.at[AT_P_LO].bin : none;
        p_hi = sh.at[AT_P_HI].bin >= 0 ? sh.at[AT_P_HI].bin : kBins - 1;
        if (p_lo != none) lo = fmin(lo, sh.at[AT_P_LO].mass_before);
        if (sh.at[AT_P_HI].bin >= 0) hi = fmin(hi, sh.at[AT_P_HI].mass_before + sh.at[AT_P_HI].mass);
    }
    if (mb != none) {
        lo = fmin(lo, sh.at[AT_M].mass_before);
        hi = fmin(hi, sh.at[AT_M].mass_before + sh.at[AT_M].mass);
    }
    hi = fmax(hi, sh.at[AT_FIRST].mass);  // (the first token is kept whatever the filters say)
    find<false>(sh, own, u * lo, AT_D_LO);
    find<false>(sh, own, u * hi, AT_D_HI);
    if (tid == 0) {
        sh.segs = 0;
        sh.listed = 0;
    }
    __syncthreads();
    const int d_lo = sh.at[AT_D_LO].bin >= 0 ? sh.at[AT_D_LO].bin : 0;
    const int d_hi = sh.at[AT_D_HI].bin >= 0 ? sh.at[AT_D_HI].bin : kBins - 1;

    // ---- their tokens, bin by bin
    auto wanted = [&](int bin) {
        return bin == kb || (bin >= p_lo && bin <= p_hi) || bin == mb || (bin >= d_lo && bin <= d_hi) || bin == first_bin;
    };
    const int own0 = tid * kOwn, own1 = own0 + kOwn - 1;
    auto near = [&](int b0, int b1) { return b0 <= own1 && b1 >= own0; };
    if (near(kb, kb) || near(p_lo, p_hi) || near(mb, mb) || near(d_lo, d_hi) || near(first_bin, first_bin))
        own.walk(sh, [&](int bin, uint64_t w, double top, int nb, double before, double) {
        if (wanted(bin)) {
            const int k = atomicAdd(&sh.segs, 1), base = atomicAdd(&sh.listed, own.count(w));
            if (k < kSegs) sh.seg[k] = Seg{before, top, own.parts(w), bin, base, own.count(w), nb, 0};
        }
    });
    __syncthreads();
    const int segs = sh.segs, listed = sh.listed;
    const bool fits = segs <= kSegs && listed <= kList;
    auto seg_of = [&](int bin) -> int {
        for (int k = 0; k < segs; ++k)
            if (sh.seg[k].bin == bin) return k;
        return -1;
    };
    Limit limit{none, 0, mass_all};
    if (fits) {
        // bins' words become their segment + 1 (0: not wanted)
        for (int j = 0; j < kOwn; ++j) sh.words[tid * kOwn + j] = 0;
        __syncthreads();
        if (tid < segs) sh.words[sh.seg[tid].bin] = tid + 1;
        __syncthreads();
        int b0 = kBins, b1 = -1;
        for (int k = 0; k < segs; ++k) {
            b0 = min(b0, sh.seg[k].bin);
            b1 = max(b1, sh.seg[k].bin);
        }
        // no logit below this reaches those bins (the margin is far above the roundings of both sides)
        const float least_v = bn.value_below(b1);
        scan_row<DT>(row, 0, a.vocab, [&](int i, float v) {
            if (!(v >= least_v)) return;
            int bin;
            double part;
            if (!bn.place(v, bin, part) || bin < b0 || bin > b1) return;
            const int k = (int)sh.words[bin] - 1;
            if (k < 0) return;
            const int slot = atomicAdd(&sh.seg[k].cursor, 1), at = sh.seg[k].base + slot;
            if (slot >= sh.seg[k].n) return;
            sh.list[at] = (uint64_t)~order_key(v) << 32 | (uint32_t)i;
            sh.list_seg[at] = (uint8_t)k;
        });
        __syncthreads();
        // ---- ranked inside their bins, with the parts before each
        uint64_t* ranked = sh.words;
        uint64_t* before = sh.words + kList;
        auto parts_of = [&](uint64_t key) -> uint64_t {
            int bin;
            double part = 0.0;
            bn.place(key_value(~(uint32_t)(key >> 32)), bin, part);
            return (uint64_t)a.q_scale - bn.q_of(part);
        };
        uint64_t* parts = sh.words + 2 * kList;            // each token's own
        uint64_t* sums = sh.words + 3 * kList;             // those of the tokens ahead of it in its bin
        uint32_t* ranks = (uint32_t*)(sh.words + 4 * kList);  // their number
        for (int i = tid; i < listed; i += kThreads) {
            parts[i] = parts_of(sh.list[i]);
            sums[i] = 0;
            ranks[i] = 0;
        }
        __syncthreads();
        // the comparisons of a bin's tokens, shared out over the threads
        const int shares = max(1, kThreads / max(listed, 1));
        for (int x = tid; x < listed * shares; x += kThreads) {
            const int i = x / shares, from = x - i * shares;
            const Seg& s = sh.seg[sh.list_seg[i]];
            const uint64_t key = sh.list[i];
            int rank = 0;
            uint64_t sum = 0;
#pragma unroll 4
            for (int j = s.base + from; j < s.base + s.n; j += shares) {
                const bool ahead = sh.list[j] < key;
                rank += ahead;
                sum += ahead ? parts[j] : 0;
            }
            if (rank) {
                atomicAdd(&ranks[i], (uint32_t)rank);
                atomicAdd((unsigned long long*)&sums[i], (unsigned long long)sum);
            }
        }
        __syncthreads();
        for (int i = tid; i < listed; i += kThreads) {
            const int to = sh.seg[sh.list_seg[i]].base + (int)ranks[i];
            ranked[to] = sh.list[i];
            before[to] = sums[i];
        }
        __syncthreads();
        auto sum_to = [&](const Seg& s, int j) -> uint64_t { return j < s.n ? before[s.base + j] : s.total; };
        auto mass_to = [&](const Seg& s, int j) -> double {
            return s.mass_before + s.top * ((double)sum_to(s, j) * a.q_unit);
        };
        // how many of a segment's tokens satisfy g(position): g is true, then false
        auto many = [&](const Seg& s, auto g) -> int {
            int lo_ = 0, hi_ = s.n;
            while (lo_ < hi_) {
                const int mid = (lo_ + hi_) >> 1;
                if (g(mid)) lo_ = mid + 1;
                else hi_ = mid;
            }
            return lo_;
        };
        double mass_k = mass_all;
        if (by_k) {
            const Seg& s = sh.seg[seg_of(kb)];
            limit = Limit{kb, top_k - s.count_before, mass_to(s, top_k - s.count_before)};
            mass_k = limit.mass;
        }
        if (by_p) {
            const double x = p_of * mass_k;
            int pick = -1;
            for (int k = 0; k < segs; ++k) {
                const Seg& s = sh.seg[k];
                if (s.bin >= p_lo && s.bin <= p_hi && mass_to(s, s.n) > x && (pick < 0 || s.bin < sh.seg[pick].bin)) pick = k;
            }
            if (pick >= 0) {
                const Seg& s = sh.seg[pick];
                const int m = max(1, many(s, [&](int j) { return mass_to(s, j) <= x; }));
                const Limit l{s.bin, m, mass_to(s, m)};
                if (l.before(limit)) limit = l;
            }
        }
        if (by_m && mb != none) {
            const int k = seg_of(mb);
            Limit l{mb, 0, sh.at[AT_M].mass_before};
            if (k >= 0) {
                const Seg& s = sh.seg[k];
                l.n = many(s, [&](int j) {
                    return s.top * ((double)(sum_to(s, j + 1) - sum_to(s, j)) * a.q_unit) >= least;
                });
                l.mass = mass_to(s, l.n);
            }
            if (l.before(limit)) limit = l;
        }
        {  // the first token is always kept
            const Seg& s = sh.seg[seg_of(first_bin)];
            const Limit one{first_bin, 1, mass_to(s, 1)};
            if (limit.before(one)) limit = one;
        }
        const double x = u * limit.mass;
        int pick = -1, last = -1;
        for (int k = 0; k < segs; ++k) {
            const Seg& s = sh.seg[k];
            if (s.bin > limit.bin || (s.bin == limit.bin && limit.n == 0)) continue;
            if (last < 0 || s.bin > sh.seg[last].bin) last = k;
            const int m = s.bin == limit.bin ? limit.n : s.n;
            if (mass_to(s, m) > x && (pick < 0 || s.bin < sh.seg[pick].bin)) pick = k;
        }
        if (pick < 0) pick = last;
        if (tid == 0) {
            const Seg& s = sh.seg[pick];
            const int m = s.bin == limit.bin ? limit.n : s.n;
            const int j = min(m - 1, many(s, [&](int i) { return mass_to(s, i + 1) <= x; }));
            a.tokens[r] = (int64_t)(uint32_t)ranked[s.base + j];
            if (a.probs)
                a.probs[r] = (float)(s.top * ((double)(sum_to(s, j + 1) - sum_to(s, j)) * a.q_unit) / limit.mass);
        }
        __syncthreads();
        return;
    }
    if constexpr (FULL)
        finish_full<DT>(a, sh, row, r, bn, u, by_k ? top_k : 0, by_p ? p_of : -1.0, least, mb, mass_all);
    else if (tid == 0) a.tokens[r] = -1;  // left to the next launch
}

// The first largest logit of the tokens [e0, e1): its order key, and its index inverted.
template <int DT>
__device__ uint64_t range_best(Shared& sh, const char* row, int e0, int e1) {
    uint64_t best = 0;
    scan_row<DT>(row, e0, e1, [&](int i, float v) {
        const uint64_t k = (uint64_t)order_key(v) << 32 | (uint32_t)~i;
        best = k > best ? k : best;
    });
    if (threadIdx.x == 0) sh.best = 0;
    __syncthreads();
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t x = __shfl_xor((unsigned long long)best, o, 64);
        best = x > best ? x : best;
    }
    if ((threadIdx.x & 63) == 0) atomicMax(&sh.best, (unsigned long long)best);
    __syncthreads();
    return sh.best;
}

template <int DT>
__device__ float range_max(Shared& sh, const char* row, int e0, int e1) {
    float m = -__builtin_huge_valf();
    scan_row<DT>(row, e0, e1, [&](int, float v) { m = fmaxf(m, v); });
    return block_max(sh, m);
}

// A row whose largest logit is infinite: its tokens of that logit (all, where it is -infinity)
// are alike, the others nothing. Every boundary is a number of them.
template <int DT>
__device__ void alike_row(const SampleArgs& a, Shared& sh, const char* row, int r, float largest) {
    const int per = (a.vocab + kThreads - 1) / kThreads;
    const int i0 = min((int)threadIdx.x * per, a.vocab), i1 = min(i0 + per, a.vocab);
    auto is = [&](int i) {
        const float v = value_of<DT>(DT == MF_F32 ? ((const uint32_t*)row)[i] : (uint32_t)((const uint16_t*)row)[i]);
        return largest < 0.f || v == largest;
    };
    int n = 0, all;
    for (int i = i0; i < i1; ++i) n += is(i);
    int before = n;
    double none = 0.0, end, sum;
    block_sums(sh, before, none, end, all, sum);
    const int top_k = a.top_k ? a.top_k[r] : a.top_k0;
    const double top_p = a.top_p ? a.top_p[r] : a.top_p0;
    const double min_p = a.min_p ? a.min_p[r] : a.min_p0;
    double u = a.uniforms[r];
    u = u > 0.0 ? fmin(u, 1.0 - 0x1p-24) : 0.0;
    int kept = top_k > 0 ? min(top_k, all) : all;
    if (!(top_p >= 1.0)) kept = min(kept, (int)floor((top_p > 0.0 ? top_p : 0.0) * kept) + 1);
    if (min_p > 1.0) kept = 1;
    int at = min((int)floor(u * kept), kept - 1) - before;
    if (at >= 0 && at < n) {
        for (int i = i0; i < i1; ++i)
            if (is(i) && at-- == 0) {
                a.tokens[r] = i;
                if (a.probs) a.probs[r] = (float)(1.0 / kept);
            }
    }
}

// The bins of a part of a row, added to the row's in memory (few rows: their parts spread over
// the GPU).
template <int DT>
__global__ __launch_bounds__(kThreads) void bins_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int r = blockIdx.y, e0 = blockIdx.x * a.chunk, e1 = min(e0 + a.chunk, a.vocab);
    const char* row = a.logits + (int64_t)r * a.stride_row * (DT == MF_F32 ? 4 : 2);
    uint64_t* out = a.bins + (int64_t)r * kRowWords;
    const float temp = a.temp ? a.temp[r] : a.temp0;
    if (!(temp > 0.f)) {
        const uint64_t best = range_best<DT>(sh, row, e0, e1);
        if (threadIdx.x == 0) atomicMax((unsigned long long*)&out[kBins], (unsigned long long)best);
        return;
    }
    clear_words(sh);
    float ref = range_max<DT>(sh, row, 0, min(a.vocab, kFirst));
    if (isinf(ref)) ref = range_max<DT>(sh, row, 0, a.vocab);
    float largest = ref;
    if (!isinf(ref)) {
        largest = bin_range<DT>(a, sh, row, Binner(a, ref, temp), e0, e1);
        for (int i = threadIdx.x; i < kBins; i += kThreads) {
            const uint64_t w = sh.words[i];
            if (w) atomicAdd((unsigned long long*)&out[i], (unsigned long long)w);
        }
    }
    if (threadIdx.x == 0) {
        atomicMax((unsigned long long*)&out[kBins], (unsigned long long)order_key(largest) << 32);
        if (blockIdx.x == 0) out[kBins + 1] = __float_as_uint(ref);
    }
}

// One workgroup a row. WHOLE: the row from its logits on. PARTS: from the bins that bins_kernel
// left, which it clears. FULL: the rows that the launch before left (token -1), because their
// boundary bins hold too many tokens or a logit lies above the bins; in a kernel of their own,
// since their code's registers made every other row's loops spill (256 rows of 130021: 127 us in
// one kernel).
enum { WHOLE, PARTS, FULL };

template <int DT, int MODE>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int r = blockIdx.x;
    if (MODE == FULL && a.tokens[r] >= 0) return;
    const char* row = a.logits + (int64_t)r * a.stride_row * (DT == MF_F32 ? 4 : 2);
    const float temp = a.temp ? a.temp[r] : a.temp0;
    if constexpr (MODE == PARTS) {
        uint64_t* in = a.bins + (int64_t)r * kRowWords;
        const uint64_t best = in[kBins];
        const float ref = __uint_as_float((uint32_t)in[kBins + 1]);
        const float largest = key_value((uint32_t)(best >> 32));
        const bool greedy = !(temp > 0.f);
        if (!greedy) {
            for (int i = threadIdx.x; i < kBins; i += kThreads) {
                const uint64_t w = in[i];
                sh.words[i] = w;
                if (w) in[i] = 0;
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) in[kBins] = in[kBins + 1] = 0;
        if (greedy) {
            if (threadIdx.x == 0) {
                a.tokens[r] = (int64_t)(uint32_t)~(uint32_t)best;
                if (a.probs) a.probs[r] = 1.f;
            }
            return;
        }
        if (!isinf(ref)) {
            const Binner bn(a, ref, temp);
            if (largest <= bn.hi) finish_row<DT, false>(a, sh, row, r, bn, largest);
            else if (threadIdx.x == 0) a.tokens[r] = -1;
            return;
        }
        alike_row<DT>(a, sh, row, r, largest);
    } else {
        if (!(temp > 0.f)) {
            const uint64_t best = range_best<DT>(sh, row, 0, a.vocab);
            if (threadIdx.x == 0) {
                a.tokens[r] = (int64_t)(uint32_t)~(uint32_t)best;
                if (a.probs) a.probs[r] = 1.f;
            }
            return;
        }
        clear_words(sh);
        float ref = range_max<DT>(sh, row, 0, min(a.vocab, kFirst));
        if (isinf(ref)) ref = range_max<DT>(sh, row, 0, a.vocab);
        float largest = ref;
        if (!isinf(ref)) {
            Binner bn(a, ref, temp);
            for (;;) {
                largest = bin_range<DT>(a, sh, row, bn, 0, a.vocab);
                if (largest <= bn.hi || isinf(largest)) break;
                bn = Binner(a, largest, temp);  // above the bins: again from the true maximum
                __syncthreads();
                clear_words(sh);
                __syncthreads();
            }
            if (!isinf(largest)) {
                finish_row<DT, MODE == FULL>(a, sh, row, r, bn, largest);
                return;
            }
        }
        alike_row<DT>(a, sh, row, r, largest);
    }
}

// Tokens of one workgroup's part, 0 where rows are not split: about num_cus / 4 parts, of at
// least 4096 tokens. More of them cost more in the memory's additions, a few thousand a part,
// than they win: us a call, unsplit, and 16, 32 and 64 parts: one row of 130021 fp32 logits 68, 50,
// 50, 50, 16 rows 69, 69, 60, 57, 32 rows 71, 71, 70, 63 (64 rows in 512 parts: 331 against 50).
int chunk_for(int num_rows, int vocab, int num_cus) {
    const int parts = std::min(num_cus / 4 / num_rows, (vocab + 4095) / 4096);
    return parts < 2 ? 0 : ((vocab + parts - 1) / parts + 7) / 8 * 8;
}

template <int DT>
int launch_sample(const SampleArgs& a, hipStream_t st) {
    const dim3 rows((unsigned)a.num_rows), threads(kThreads);
    if (a.chunk > 0) {
        const dim3 parts((unsigned)((a.vocab + a.chunk - 1) / a.chunk), (unsigned)a.num_rows);
        hipLaunchKernelGGL((bins_kernel<DT>), parts, threads, 0, st, a);
        if (int e = check_launch()) return e;
        hipLaunchKernelGGL((sample_kernel<DT, PARTS>), rows, threads, 0, st, a);
    } else {
        hipLaunchKernelGGL((sample_kernel<DT, WHOLE>), rows, threads, 0, st, a);
    }
    if (int e = check_launch()) return e;
    hipLaunchKernelGGL((sample_kernel<DT, FULL>), rows, threads, 0, st, a);
    return check_launch();
}

}  // namespace
}  // namespace mf

extern "C" int64_t mf_sample_workspace_size(int num_rows, int vocab, int num_cus) {
    using namespace mf;
    if (num_rows < 1 || vocab < 1 || vocab > MF_SAMPLE_MAX_VOCAB || num_cus < 1) return 0;
    return chunk_for(num_rows, vocab, num_cus) > 0 ? (int64_t)num_rows * kRowWords * 8 : 0;
}

extern "C" int mf_sample(const void* logits, int dtype, int64_t stride_row, int num_rows, int vocab,
                         const float* uniforms, const float* temperature, float temperature0, const int32_t* top_k,
                         int top_k0, const float* top_p, float top_p0, const float* min_p, float min_p0,
                         int64_t* tokens, float* probs, int num_cus, void* workspace, int64_t workspace_bytes,
                         mf_stream_t stream) {
    using namespace mf;
    if (!dtype_ok(dtype) || num_cus < 1 || num_rows < 0 || vocab < 1 || vocab > MF_SAMPLE_MAX_VOCAB || stride_row < 0) return MF_ERR_ARG;
    if (num_rows == 0) return MF_OK;
    if (!logits || !uniforms || !tokens || ((uintptr_t)workspace & 7)) return MF_ERR_ARG;
    const int64_t need = mf_sample_workspace_size(num_rows, vocab, num_cus);
    if (need > 0 && (!workspace || workspace_bytes < need)) return MF_ERR_WORKSPACE;
    int lv = 0;
    while ((1 << lv) < vocab) ++lv;
    const int qs = std::min(40, 71 - 2 * lv);
    SampleArgs a{(const char*)logits, stride_row, vocab, num_rows, uniforms, temperature, top_k, top_p, min_p,
                 temperature0, top_p0, min_p0, top_k0, 63 - lv, (double)(1ull << qs), 1.0 / (double)(1ull << qs),
                 tokens, probs, (uint64_t*)workspace, need > 0 ? chunk_for(num_rows, vocab, num_cus) : 0};
    static_assert(sizeof(Shared) <= 160 * 1024, "LDS of one compute unit");
    hipStream_t st = (hipStream_t)stream;
    if (dtype == MF_F32) return launch_sample<MF_F32>(a, st);
    if (dtype == MF_F16) return launch_sample<MF_F16>(a, st);
    return launch_sample<MF_BF16>(a, st);
}
