// fm_logprob.hip — log probability of a given token, entropy and the largest alternatives of rows
// of logits (include/finch_hip.h, fm_logprobs_dev), in one pass over the logits.
//
// A row is cut into segments of FM_LP_SEG elements, one workgroup each, sixteen elements a thread in
// registers.  With d_i = x_i - m, m the row's maximum and the (first) maximum's own term e^0 = 1
// kept apart,
//   Z' = sum over the others of e^d,  log p_i = d_i - log1p(Z'),  H = log1p(Z') - sum e^d d / (1 + Z')
// so that neither loses its digits when one token holds nearly all the probability.  A segment
// gives (m, Z', sum e^d d) for its own maximum, and its top_n largest elements.
//
// Order: an element's key is its value, made an unsigned number of the same order, above the complement
// of its index: keys of a row are distinct, and the larger key is the larger value or, of equal
// ones, the lower index.  The top_n keys of a segment: the top_n-th largest of the threads'
// maxima bounds the top_n-th largest key from below, and at most 16 top_n keys (those of top_n threads)
// are not below it; they are ranked by counting.  The second kernel joins a row's segments the same way.
#include "fm_common.h"

namespace {

constexpr int LP_T = 256, LP_E = 16;           // threads, elements per thread
constexpr int LP_SEG = LP_T * LP_E;
constexpr int LP_TOP = 32;

typedef unsigned long long LpKey;

__device__ __forceinline__ uint32_t order_bits(float x) {      // unsigned order of the floats
    const uint32_t b = __float_as_uint(x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
// -0 and +0 are equal values: both take the key of +0
__device__ __forceinline__ LpKey make_key(float x, uint32_t idx) {
    return (LpKey)order_bits(x == 0.0f ? 0.0f : x) << 32 | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ LpKey key_max(LpKey a, LpKey b) { return a > b ? a : b; }

struct Part {             // what a segment leaves: statistics relative to its own maximum
    float m, z, ed;       // maximum, sum of e^d without the maximum's own term, sum of e^d d
    int bad;              // holds a NaN or +inf
};

struct Shared {
    LpKey keys[LP_T];
    LpKey cand[LP_E * LP_TOP];
    LpKey bound;
    float red[2][LP_T / 64];
    int n_cand;
};

// The n largest of the block's keys (E per thread; key 0 = none) into dst[0..n), largest first,
// 0 where there are fewer.  mine: the thread's largest key.
template <int E>
__device__ __forceinline__ void block_top(const LpKey *k, LpKey mine, int n, Shared &sh, LpKey *dst) {
    const int t = threadIdx.x;
    sh.keys[t] = mine;
    if (t == 0) sh.n_cand = 0, sh.bound = 0;
    __syncthreads();
    // the thread's place among the threads' maxima: the first n threads hold all candidates
    int place = 0;
    for (int j = 0; j < LP_T; j++) place += sh.keys[j] > mine;
    // (keys are distinct but for the empty key 0; with fewer than n keys the bound stays 0)
    if (place == n - 1) sh.bound = mine;
    __syncthreads();
    const LpKey bound = sh.bound;
    if (mine >= bound && mine) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (k[e] >= bound && k[e]) {
                const int at = atomicAdd(&sh.n_cand, 1);
                if (at < LP_E * LP_TOP) sh.cand[at] = k[e];
            }
    }
    __syncthreads();
    const int c = min(sh.n_cand, LP_E * LP_TOP);
    for (int i = t; i < c; i += LP_T) {
        const LpKey v = sh.cand[i];
        int rank = 0;
        for (int j = 0; j < c; j++) rank += sh.cand[j] > v;
        if (rank < n) dst[rank] = v;
    }
    for (int i = c + t; i < n; i += LP_T) dst[i] = 0;
}

__global__ __launch_bounds__(LP_T) void fm_logprob_seg(const float *x, int vocab, int64_t stride, int n_seg, int top_n,
                                                       Part *parts, LpKey *tops) {
    __shared__ Shared sh;
    __shared__ LpKey wmax[LP_T / 64];
    const int row = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const float *r = x + (int64_t)row * stride;
    const int base = seg * LP_SEG;
    float v[LP_E];
    LpKey k[LP_E], mine = 0;
    int bad = 0;
#pragma unroll
    for (int e = 0; e < LP_E; e++) {
        const int i = base + e * LP_T + t;
        v[e] = i < vocab ? r[i] : -INFINITY;
        k[e] = i < vocab ? make_key(v[e], (uint32_t)i) : 0;
        bad |= i < vocab && !(v[e] < INFINITY);
        mine = key_max(mine, k[e]);
    }
    LpKey top = mine;
    for (int o = 32; o; o >>= 1) top = key_max(top, (LpKey)__shfl_xor((unsigned long long)top, o));
    if ((t & 63) == 0) wmax[t >> 6] = top;
    bad = __syncthreads_or(bad);
    for (int w = 0; w < LP_T / 64; w++) top = key_max(top, wmax[w]);
    const float m = from_order((uint32_t)(top >> 32));
    float z = 0.0f, ed = 0.0f;
    if (!bad && m > -INFINITY) {
#pragma unroll
        for (int e = 0; e < LP_E; e++) {
            const float d = v[e] - m, p = expf(d);
            if (k[e] != top && p > 0.0f) {     // (0 * -inf must not come in)
                z += p;
                ed = fmaf(p, d, ed);
            }
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
        p.bad = bad;
        parts[(size_t)row * n_seg + seg] = p;
    }
    if (top_n) block_top<LP_E>(k, mine, top_n, sh, tops + ((size_t)row * n_seg + seg) * top_n);
}

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
    float m = -INFINITY;
    int bad = 0;
    for (int i = t; i < n_seg; i += LP_T) m = fmaxf(m, p[i].m), bad |= p[i].bad;
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) stat[wave] = m;
    bad = __syncthreads_or(bad);
    m = fmaxf(fmaxf(stat[0], stat[1]), fmaxf(stat[2], stat[3]));
    __syncthreads();
    // the first segment that holds the maximum keeps its own 1 apart, the others' ones count
    int first = n_seg;
    for (int i = t; i < n_seg; i += LP_T)
        if (p[i].m == m) first = min(first, i);
    for (int o = 32; o; o >>= 1) first = min(first, __shfl_xor(first, o));
    if (lane == 0) stat[wave] = __int_as_float(first);
    __syncthreads();
    first = min(min(__float_as_int(stat[0]), __float_as_int(stat[1])), min(__float_as_int(stat[2]), __float_as_int(stat[3])));
    float z = 0.0f, ed = 0.0f;
    if (!bad && m > -INFINITY)
        for (int i = t; i < n_seg; i += LP_T) {
            const float d = p[i].m - m, one = i == first ? 0.0f : 1.0f;
            const float e = expf(d);
            if (!(e > 0.0f)) continue;         // (0 * -inf must not come in)
            z = fmaf(e, p[i].z + one, z);
            // sum e^(d_i + d) (d_i + d) over the segment's elements
            ed += e * (p[i].ed + d * (p[i].z + one));
        }
    z = fm_group_sum<64>(z);
    ed = fm_group_sum<64>(ed);
    if (lane == 0) sh.red[0][wave] = z, sh.red[1][wave] = ed;
    __syncthreads();
    if (t == 0) {
        z = ((sh.red[0][0] + sh.red[0][1]) + sh.red[0][2]) + sh.red[0][3];
        ed = ((sh.red[1][0] + sh.red[1][1]) + sh.red[1][2]) + sh.red[1][3];
        const float logz = log1pf(z);
        const bool none = !(m > -INFINITY);
        if (entropy) entropy[row] = bad ? NAN : none ? 0.0f : logz - ed / (1.0f + z);
        if (logprob) {
            const int id = tokens[row];
            float lp = -INFINITY;
            if (bad) lp = NAN;
            else if (id >= 0 && id < vocab && !none) lp = (x[(int64_t)row * stride + id] - m) - logz;
            logprob[row] = lp;
        }
        s_m = none ? 0.0f : m;
        s_logz = logz;
    }
    __syncthreads();
    if (!top_n) return;
    // the segments' lists: few enough keys for one thread to keep its own (vocab < 2^31)
    const LpKey *src = tops + (size_t)row * n_seg * top_n;
    const int total = n_seg * top_n;
    LpKey bound_keys[LP_E];
    // rounds of LP_SEG keys, the best so far riding along
    for (int i = t; i < LP_TOP; i += LP_T) best[i] = 0;
    __syncthreads();
    for (int at = 0; at < total; at += LP_SEG - LP_TOP) {
        LpKey mine = 0;
#pragma unroll
        for (int e = 0; e < LP_E; e++) {
            const int i = e * LP_T + t;
            LpKey kk = 0;
            if (i < LP_TOP) kk = i < top_n ? best[i] : 0;
            else if (at + i - LP_TOP < total) kk = src[at + i - LP_TOP];
            bound_keys[e] = kk;
            mine = key_max(mine, kk);
        }
        __syncthreads();
        block_top<LP_E>(bound_keys, mine, top_n, sh, best);
        __syncthreads();
    }
    if (t < top_n) {
        const LpKey kk = best[t];
        const float v = from_order((uint32_t)(kk >> 32));
        ids[(size_t)row * top_n + t] = bad ? -1 : (int32_t)(0xFFFFFFFFu - (uint32_t)kk);
        top_lp[(size_t)row * top_n + t] = bad ? NAN : (v - s_m) - s_logz;
    }
}

}  // namespace

extern "C" size_t fm_logprob_ws(int rows, int vocab, int top_n) {
    const size_t n_seg = ((size_t)vocab + LP_SEG - 1) / LP_SEG;
    return (size_t)rows * n_seg * (sizeof(Part) + (size_t)top_n * sizeof(LpKey));
}

extern "C" int fm_launch_logprob(const float *x, int rows, int vocab, int64_t stride, const int32_t *tokens, int top_n,
                                 float *logprob, float *entropy, int32_t *ids, float *top_lp, void *ws, hipStream_t st) {
    const int n_seg = (int)(((int64_t)vocab + LP_SEG - 1) / LP_SEG);
    LpKey *tops = (LpKey *)ws;
    Part *parts = (Part *)(tops + (size_t)rows * n_seg * top_n);
    hipLaunchKernelGGL(fm_logprob_seg, dim3(n_seg, rows), dim3(LP_T), 0, st, x, vocab, stride, n_seg, top_n, parts, tops);
    hipLaunchKernelGGL(fm_logprob_join, dim3(rows), dim3(LP_T), 0, st, x, vocab, stride, n_seg, top_n, parts, tops, tokens,
                       logprob, entropy, ids, top_lp);
    return hipGetLastError() == hipSuccess ? FM_OK : FM_ERR_HIP;
}
