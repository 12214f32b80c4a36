// fm_logprob.hip — log probability of a given token, entropy and the largest alternatives of rows
// of logits (include/finch_hip.h, fm_logprobs_dev), in one pass over the logits.
//
// A row is cut into segments, one workgroup each, E elements a thread in registers.  With d_i = x_i - m,
// m the row's maximum and the (first) maximum's own term e^0 = 1 kept apart,
//   Z' = sum over the others of e^d,  log p_i = d_i - log1p(Z'),  H = log1p(Z') - sum e^d d / (1 + Z')
// so that neither loses its digits when one token holds nearly all the probability.  (e^d is the instruction's 2^x of
// d log2 e in fp32: with half of the probability 10 to 20 below the maximum the mean error of log p is 1.7e-8 at 0.69,
// a quarter of a step, and that of the entropy 7.9e-8 at 6.2, a sixth.)  A segment
// gives (m, Z', sum e^d d) for its own maximum, and its top_n largest elements.
//
// Order: an element's key is its value, made an unsigned number of the same order, above the complement
// of its index: keys of a row are distinct, and the larger key is the larger value or, of equal
// ones, the lower index.  The top_n keys of a segment: the top_n-th largest of a wave's 64 lane
// maxima (to 16 bits, found bit by bit with ballots) bounds the segment's top_n-th value from below, so
// does the largest of the waves' bounds; the elements that reach it, few more than top_n, are
// collected, a list a wave, and ranked by counting.  (Equal values, or many of the largest in one lane, may be
// more than there is room for: then the maximum is taken top_n times instead.)  A second kernel joins a row's
// segments the same way.
//
// 257 rows of 248320, top 5: 53 us, 4.8 TB/s, the rate of a large copy: bound by the loads and, close behind, by
// the vector ALU (ten instruction slots an element, four of them the exponential's).  One row, top 20: 13.7 us,
// the latency of two kernels, 8.8 of it without alternatives.
#include "fm_common.h"

namespace {

constexpr int LP_T = 256;            // threads
constexpr int LP_TOP = 32;
constexpr int LP_LIST = 128;         // candidates a wave has room for

typedef unsigned long long LpKey;
typedef float fm_v4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ uint32_t order_bits(float x) {      // unsigned order of the floats
    // (-0 and +0 are equal values: both take the place of +0)
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float from_order(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ LpKey make_key(float x, uint32_t idx) {
    return (LpKey)order_bits(x) << 32 | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ LpKey key_max(LpKey a, LpKey b) { return a > b ? a : b; }
__device__ __forceinline__ LpKey wave_key_max(LpKey k) {
    for (int o = 32; o; o >>= 1) k = key_max(k, (LpKey)__shfl_xor(k, o));
    return k;
}

struct Part {             // what a segment leaves: statistics relative to its own maximum
    float m, z, ed;       // maximum, sum of e^d without the maximum's own term, sum of e^d d
    int bad;              // holds a NaN or +inf
};

struct Shared {
    LpKey cand[LP_T / 64][LP_LIST + 2], bound[LP_T / 64];   // (lists four banks apart)
    float red[2][LP_T / 64];
    int n_cand[LP_T / 64];
};

// The largest t with zero low half that at least n of the wave's lanes reach; 0 if fewer than n lanes have one.
__device__ __forceinline__ uint32_t nth_largest(uint32_t v, int n) {
    uint32_t t = 0;
#pragma unroll
    for (int b = 31; b >= 16; b--) {
        const uint32_t trial = t | 1u << b;
        if (__popcll(__ballot(v >= trial)) >= n) t = trial;
    }
    return t;
}

// The n largest of the block's keys into dst[0..n), largest first, 0 where there are fewer.  key(e), e < E:
// the thread's e-th (0 = none); reaches(e, bound): whether its value's order bits may reach the bound;
// big: the largest of those.
template <int E, class Key, class Reaches>
__device__ __forceinline__ void block_top(Key key, Reaches reaches, uint32_t big, int n, Shared &sh, LpKey *dst) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const uint32_t of_wave = nth_largest(big, n);
    if (lane == 0) sh.bound[wave] = of_wave;
    __syncthreads();
    uint32_t bound = 1;      // (order bits are never 0 for a number: 0 marks "none")
#pragma unroll
    for (int w = 0; w < LP_T / 64; w++) bound = max(bound, (uint32_t)sh.bound[w]);
    int c = 0;
    if (__ballot(big >= bound)) {
#pragma unroll
        for (int e = 0; e < E; e++) {
            const bool in = reaches(e, bound);
            if (!__ballot(in)) continue;
            const LpKey k = in ? key(e) : (LpKey)0;
            const unsigned long long mask = __ballot(k != 0);
            const int at = c + __popcll(mask & ((1ull << lane) - 1));
            if (k && at < LP_LIST) sh.cand[wave][at] = k;
            c += __popcll(mask);
        }
    }
    if (lane == 0) sh.n_cand[wave] = c;
    __syncthreads();
    static_assert(LP_T == 256, "four lists");
    const int c0 = sh.n_cand[0], c1 = c0 + sh.n_cand[1], c2 = c1 + sh.n_cand[2], all = c2 + sh.n_cand[3];
    if (max(max(c0, c1 - c0), max(c2 - c1, all - c2)) <= LP_LIST) {
        // four lanes a candidate, each counts the larger ones of one list
        const LpKey *list = sh.cand[t & 3];
        const int many = sh.n_cand[t & 3];
        for (int i = t >> 2; i < all; i += LP_T / 4) {
            const LpKey v = i < c0 ? sh.cand[0][i] : i < c1 ? sh.cand[1][i - c0] : i < c2 ? sh.cand[2][i - c1] : sh.cand[3][i - c2];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < many; j++) rank += list[j] > v;
            rank += __shfl_xor(rank, 1);
            rank += __shfl_xor(rank, 2);
            if (!(t & 3) && rank < n) dst[rank] = v;
        }
        for (int i = all + t; i < n; i += LP_T) dst[i] = 0;
        return;
    }
    LpKey below = ~0ull;
    for (int i = 0; i < n; i++) {
        LpKey best = 0;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const LpKey k = key(e);
            if (k < below) best = key_max(best, k);
        }
        best = wave_key_max(best);
        __syncthreads();                       // (the last round's values have been read)
        if ((t & 63) == 0) sh.bound[t >> 6] = best;
        __syncthreads();
        below = 0;
#pragma unroll
        for (int w = 0; w < LP_T / 64; w++) below = key_max(below, sh.bound[w]);
        if (t == 0) dst[i] = below;
    }
}

// V4: rows are 16-byte aligned, a thread takes four elements side by side
// (Five waves a SIMD: 257 rows 53 us, 14 registers spilled with E 32; the 99 the compiler would take leave four, 57 us, and
// for six more are spilled, 55 us.)
template <int E, bool V4>
__global__ __launch_bounds__(LP_T, 5) void fm_logprob_seg(const float *x, int vocab, int64_t stride, int n_seg, int top_n,
                                                       Part *parts, LpKey *tops) {
    __shared__ Shared sh;
    const int row = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const float *r = x + (int64_t)row * stride;
    const int base = seg * (LP_T * E);
    auto index = [&](int e) { return V4 ? base + (e >> 2) * (4 * LP_T) + 4 * t + (e & 3) : base + e * LP_T + t; };
    float v[E];
    if (base + LP_T * E <= vocab) {
#pragma unroll
        for (int e = 0; e < E; e += V4 ? 4 : 1) {
            if constexpr (V4) {
                const fm_v4 w = __builtin_nontemporal_load((const fm_v4 *)(r + index(e)));
                v[e] = w[0], v[e + 1] = w[1], v[e + 2] = w[2], v[e + 3] = w[3];
            } else {
                v[e] = __builtin_nontemporal_load(r + index(e));
            }
        }
    } else {               // the row's last segment
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = r[min(index(e), vocab - 1)];
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = index(e) < vocab ? v[e] : -INFINITY;
    }
    float big = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int e = 0; e < E; e++) bad |= !(v[e] < INFINITY), big = fmaxf(big, v[e]);
    float m = big;
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if ((t & 63) == 0) sh.red[0][t >> 6] = m;
    const bool any_bad = __syncthreads_or(bad);
    m = fmaxf(fmaxf(sh.red[0][0], sh.red[0][1]), fmaxf(sh.red[0][2], sh.red[0][3]));
    __syncthreads();
    // The maximum's own term is left out: of the first thread's first element that has it.  (Which of equal ones
    // does not matter: their terms are the same.)
    const unsigned long long have = __ballot(big == m);
    int owner = have ? __ffsll(have) - 1 + (t & ~63) : LP_T;
    if ((t & 63) == 0) sh.red[1][t >> 6] = __int_as_float(owner);
    __syncthreads();
    owner = min(min(__float_as_int(sh.red[1][0]), __float_as_int(sh.red[1][1])), min(__float_as_int(sh.red[1][2]), __float_as_int(sh.red[1][3])));
    __syncthreads();
    float z = 0.0f, ed = 0.0f;
    if (!any_bad && m > -INFINITY) {
        bool out = t == owner;
        const bool mine = __ballot(out) != 0;     // (this wave holds the owner)
#pragma unroll
        for (int e = 0; e < E; e++) {
            // e^-200 is 0 in fp32, and 0 * -inf must not come in
            const float d = fmaxf(v[e] - m, -200.0f);
            float p = __expf(d);
            if (mine) {
                const bool drop = out && d == 0.0f;
                p = drop ? 0.0f : p;
                out = out && !drop;
            }
            z += p;
            ed = fmaf(p, d, ed);
        }
    }
    z = fm_group_sum<64>(z);
    ed = fm_group_sum<64>(ed);
    if ((t & 63) == 0) sh.red[0][t >> 6] = z, sh.red[1][t >> 6] = ed;
    __syncthreads();
    if (t == 0) {
        Part p;
        p.m = m;
        p.z = ((sh.red[0][0] + sh.red[0][1]) + sh.red[0][2]) + sh.red[0][3];
        p.ed = ((sh.red[1][0] + sh.red[1][1]) + sh.red[1][2]) + sh.red[1][3];
        p.bad = any_bad;
        parts[(size_t)row * n_seg + seg] = p;
    }
    if (top_n) {
        // (compared as numbers: bounds below -inf stand for everything)
        auto reaches = [&](int e, uint32_t bound) { return v[e] >= (bound > 0x007FFFFFu ? from_order(bound) : -INFINITY); };
        block_top<E>([&](int e) { return index(e) < vocab ? make_key(v[e], (uint32_t)index(e)) : (LpKey)0; }, reaches,
                     index(0) < vocab ? order_bits(big) : 0u, top_n, sh, tops + ((size_t)row * n_seg + seg) * top_n);
    }
}

constexpr int JOIN_E = 8;

// joins a row's segments; one workgroup per row
__global__ __launch_bounds__(LP_T) void fm_logprob_join(const float *x, int vocab, int64_t stride, int n_seg, int top_n,
                                                        const Part *parts, const LpKey *tops, const int32_t *tokens,
                                                        float *logprob, float *entropy, int32_t *ids, float *top_lp) {
    __shared__ Shared sh;
    __shared__ LpKey best[LP_TOP];
    __shared__ float stat[LP_T / 64];
    __shared__ float s_m, s_logz;
    const int row = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const Part *p = parts + (size_t)row * n_seg;
    const LpKey *src = tops + (size_t)row * n_seg * top_n;
    const int total = n_seg * top_n;
    // what most rows need (256 segments, a round of keys, the token's logit) is requested at once
    const Part none = {-INFINITY, 0.0f, 0.0f, 0};
    const Part p0 = t < n_seg ? p[t] : none;
    LpKey k[JOIN_E];
    if (t < LP_TOP) best[t] = 0;
    auto fetch = [&](int at) {
#pragma unroll
        for (int e = 0; e < JOIN_E; e++) {
            const int i = at + e * LP_T + t - LP_TOP;
            k[e] = e * LP_T + t >= LP_TOP && i < total ? src[i] : 0;
        }
    };
    if (top_n) fetch(0);
    const int id = logprob ? tokens[row] : 0;
    const float given = logprob && id >= 0 && id < vocab ? x[(int64_t)row * stride + id] : -INFINITY;
    float m = p0.m;
    int bad = p0.bad;
    for (int i = t + LP_T; i < n_seg; i += LP_T) m = fmaxf(m, p[i].m), bad |= p[i].bad;
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) stat[wave] = m;
    bad = __syncthreads_or(bad);
    m = fmaxf(fmaxf(stat[0], stat[1]), fmaxf(stat[2], stat[3]));
    __syncthreads();
    // the first segment that holds the maximum keeps its own 1 apart, the others' ones count
    int first = p0.m == m ? t : n_seg;
    for (int i = t + LP_T; i < n_seg; i += LP_T)
        if (p[i].m == m) first = min(first, i);
    for (int o = 32; o; o >>= 1) first = min(first, __shfl_xor(first, o));
    if (lane == 0) stat[wave] = __int_as_float(first);
    __syncthreads();
    first = min(min(__float_as_int(stat[0]), __float_as_int(stat[1])), min(__float_as_int(stat[2]), __float_as_int(stat[3])));
    float z = 0.0f, ed = 0.0f;
    if (!bad && m > -INFINITY)
        for (int i = t; i < n_seg; i += LP_T) {
            const Part q = i == t ? p0 : p[i];
            const float d = q.m - m, one = i == first ? 0.0f : 1.0f;
            const float e = expf(d);
            if (!(e > 0.0f)) continue;         // (0 * -inf must not come in)
            z = fmaf(e, q.z + one, z);
            // sum e^(d_i + d) (d_i + d) over the segment's elements
            ed += e * (q.ed + d * (q.z + one));
        }
    z = fm_group_sum<64>(z);
    ed = fm_group_sum<64>(ed);
    if (lane == 0) sh.red[0][wave] = z, sh.red[1][wave] = ed;
    __syncthreads();
    if (t == 0) {
        z = ((sh.red[0][0] + sh.red[0][1]) + sh.red[0][2]) + sh.red[0][3];
        ed = ((sh.red[1][0] + sh.red[1][1]) + sh.red[1][2]) + sh.red[1][3];
        const float logz = log1pf(z);
        const bool none_seen = !(m > -INFINITY);
        if (entropy) entropy[row] = bad ? NAN : none_seen ? 0.0f : logz - ed / (1.0f + z);
        if (logprob) {
            float lp = -INFINITY;
            if (bad) lp = NAN;
            else if (!none_seen) lp = (given - m) - logz;
            logprob[row] = lp;
        }
        s_m = none_seen ? 0.0f : m;
        s_logz = logz;
    }
    if (!top_n) return;
    // the segments' lists in rounds, the best so far riding along in the first threads' first place
    __syncthreads();
    for (int at = 0; at < total; at += LP_T * JOIN_E - LP_TOP) {
        if (at) fetch(at);
        if (t < LP_TOP) k[0] = t < top_n ? best[t] : 0;
        LpKey mine = 0;
#pragma unroll
        for (int e = 0; e < JOIN_E; e++) mine = key_max(mine, k[e]);
        __syncthreads();
        block_top<JOIN_E>([&](int e) { return k[e]; }, [&](int e, uint32_t bound) { return (uint32_t)(k[e] >> 32) >= bound; }, (uint32_t)(mine >> 32), top_n,
                          sh, best);
        __syncthreads();
    }
    if (t < top_n) {
        const LpKey kk = best[t];
        const float v = from_order((uint32_t)(kk >> 32));
        ids[(size_t)row * top_n + t] = bad ? -1 : (int32_t)(0xFFFFFFFFu - (uint32_t)kk);
        top_lp[(size_t)row * top_n + t] = bad ? NAN : (v - s_m) - s_logz;
    }
}

// Elements per thread: 32 when that still gives every CU three workgroups (the selection of the
// largest runs once per segment), 16 otherwise.  Rows of 248320, top 20, with 32 / 16: 4 rows 15.0 / 13.8 us,
// 16 rows 16.3 / 16.3, 24 rows 17.6 / 18.3, 32 rows 19.4 / 21.3, 128 rows 44.4 / 45.8; top 5: 24 rows
// 13.8 / 13.6, 32 rows 14.9 / 15.4.
int per_thread(int rows, int vocab, int n_cu) {
    const int64_t segs = ((int64_t)vocab + LP_T * 32 - 1) / (LP_T * 32);
    return rows * segs >= 3 * n_cu ? 32 : 16;
}

}  // namespace

extern "C" size_t fm_logprob_ws(int rows, int vocab, int top_n) {
    const size_t n_seg = ((size_t)vocab + LP_T * 16 - 1) / (LP_T * 16);
    return (size_t)rows * n_seg * (sizeof(Part) + (size_t)top_n * sizeof(LpKey));
}

extern "C" int fm_launch_logprob(const float *x, int rows, int vocab, int64_t stride, const int32_t *tokens, int top_n,
                                 float *logprob, float *entropy, int32_t *ids, float *top_lp, void *ws, int n_cu, hipStream_t st) {
    const int E = per_thread(rows, vocab, n_cu);
    const int n_seg = (vocab + LP_T * E - 1) / (LP_T * E);
    LpKey *tops = (LpKey *)ws;
    Part *parts = (Part *)(tops + (size_t)rows * n_seg * top_n);
    const bool v4 = ((uintptr_t)x & 15) == 0 && (stride & 3) == 0;
#define FM_LP(EE, VV) \
    hipLaunchKernelGGL((fm_logprob_seg<EE, VV>), dim3(n_seg, rows), dim3(LP_T), 0, st, x, vocab, stride, n_seg, top_n, parts, tops)
    if (E == 32 && v4) FM_LP(32, true);
    else if (E == 32) FM_LP(32, false);
    else if (v4) FM_LP(16, true);
    else FM_LP(16, false);
#undef FM_LP
    hipLaunchKernelGGL(fm_logprob_join, dim3(rows), dim3(LP_T), 0, st, x, vocab, stride, n_seg, top_n, parts, tops, tokens,
                       logprob, entropy, ids, top_lp);
    return hipGetLastError() == hipSuccess ? FM_OK : FM_ERR_HIP;
}
