// fm_attn.hip — a paged cache of keys and values in 8 bits and the attention that reads it
// (include/finch_hip.h, fm_kv_append_dev / fm_kv_read_dev / fm_attn_dev).
//
// Codes are signed bytes with one scale per page and head, K as [token][dim], V as [dim][token].
//
// ---- the two products on the matrix cores ------------------------------------------------------
// A wave works on 64 keys at a time and on up to 16 columns, a column being one (row, query head)
// of the cache head.  Both products are v_mfma_f32_16x16x32_f16:
//   S^T = K q^T      A = K (16 keys x 32 dims), B = q^T (32 dims x 16 columns)
//   o^T += V^T p^T   A = V^T (16 dims x 32 keys), B = p^T (32 keys x 16 columns)
// A code is exact in fp16: 0x64 above the byte c ^ 0x80 is the number 1024 + c + 128, and one
// packed subtraction of 1152 leaves c.  The instruction's k index is only a pairing of A with B, so
// it is assigned where the operands lie: key r of tile t is key 16 (r / 4) + 4 t + r % 4 of the 64.
// Then the lanes that hold a column's scores (lane = 16 g + column; tile t, register i: key
// 16 g + 4 t + i) are those that need them as B of the second product, whose A is 16 consecutive bytes
// of a V row, and nothing moves between lanes but the column's maximum.  Every load is 16 bytes
// straight into registers.
// q and p are split in fp16 pieces behind a power of two that puts a column's largest element
// near 2^8 (2^14 for p, whose keys' value scales ride along), far above the subnormals: q in two pieces (22 bits)
// for fp32 vectors, in one for bf16 ones, which it holds exactly; p in two pieces for either (one piece's 11 bits are
// an error of 2^-12 of a weight: where the values cancel, percents of a bf16 result).
#include "fm_mix.h"

namespace {

constexpr int BK = FM_ATTN_KEYS, COLS = FM_ATTN_COLS;
constexpr float P_SHIFT = 14.0f;   // p is computed as 2^14 p
constexpr int WP = 2;              // pieces of p

__device__ __forceinline__ fm_v4f mfma(fm_v8h a, fm_v8h b, fm_v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// 2^x; below -126 (of which nothing is left in what follows) 0
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// A key's weight behind its power of two.  (The difference first: 14 - base would be rounded at the size of the scores, and
// from 2^25 on p could pass fp16's largest number.)
__device__ __forceinline__ float weight(float score, float base) { return fast_exp2((score - base) + P_SHIFT); }

// f as NP fp16 pieces whose sum it is (to 11 bits each).  With two, f has to be one fp32 value: fused with the
// product in front of it, the conversion and the remainder could round to different first pieces.
template <int NP>
__device__ __forceinline__ void split(float f, _Float16 *piece) {
    if constexpr (NP > 1) asm("" : "+v"(f));
#pragma unroll
    for (int p = 0; p < NP; p++) {
        piece[p] = (_Float16)f;
        f -= (float)piece[p];
    }
}

// The largest of a column's four lanes, in all of them.  (A swap with itself leaves either half in both: no way
// through LDS as with a shuffle, whose latency two waves a SIMD do not cover.)
__device__ __forceinline__ float column_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ int column_max(int x) {
    auto a = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
    x = max((int)a[0], (int)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
    return max((int)b[0], (int)b[1]);
}

// Powers of two.  An output is held in units of 2^ref, above every weight times value scale so far: what a key
// counts for goes by both, and a page of large values with next to no weight must not push the others below fp16.
// NO_REF: of nothing seen.
constexpr int NO_REF = -2000;
// of a step: `top` the largest of the lane's scores, `base` the column's maximum.  (At most 120 below the page's own scale,
// so that the scale in units of 2^ref stays in fp32's range; -246 of keys that are not seen, below all others.)
__device__ __forceinline__ int ref_of(float v_scale, float top, float base) {
    return (int)(__float_as_uint(v_scale) >> 23 & 255) - 126 + (int)ceilf(fmaxf(top - base, -120.0f));
}
// what is left of 2^ref when the maximum rises from m to base
__device__ __forceinline__ int ref_falls(int ref, float m, float base) {
    return max(ref + (int)ceilf(fmaxf(m - base, -1000.0f)), NO_REF);
}
// the power of two that a row's largest element is taken to 2^8 by, and back (the ends: zeros, infinities)
__device__ __forceinline__ int q_power(float big) {
    const int e = (int)(__float_as_uint(big) >> 23 & 255) - 127 - 8;
    return e < -126 ? -126 : e > 119 ? 119 : e;
}
__device__ __forceinline__ float power2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ fm_v4f times_power2(fm_v4f x, int e) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = ldexpf(x[i], e);
    return x;
}

// eight signed bytes as fp16 numbers
__device__ __forceinline__ fm_v8h codes_f16(uint32_t lo, uint32_t hi) {
    const fm_v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo ^= 0x80808080u;
    hi ^= 0x80808080u;
    union { uint32_t u[4]; fm_v8h h; fm_v2h p[4]; } r;
    r.u[0] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04010400u);
    r.u[1] = __builtin_amdgcn_perm(0x64646464u, lo, 0x04030402u);
    r.u[2] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04010400u);
    r.u[3] = __builtin_amdgcn_perm(0x64646464u, hi, 0x04030402u);
#pragma unroll
    for (int i = 0; i < 4; i++) r.p[i] = r.p[i] - off;
    return r.h;
}

// The pages of a lane's two runs of 16 keys: that of the tile rows it loads (run r / 4) and that of its
// scores and of V (run g).  The table is read on every path and a step ahead, its entry checked when it
// is used: whoever looks at a load's result waits for all that were issued before it.
struct Runs {
    int k, v;        // table entries
    __device__ __forceinline__ void load(const FmKv &c, const int32_t *table, int pos0) {
        const int lane = threadIdx.x & 63;
        k = table[min((pos0 + 16 * ((lane & 15) >> 2)) >> c.page_shift, c.max_pages - 1)];
        v = table[min((pos0 + 16 * (lane >> 4)) >> c.page_shift, c.max_pages - 1)];
    }
    // page, or -1 for one that is not there
    static __device__ __forceinline__ int checked(const FmKv &c, int entry, int pos) {
        return (pos >> c.page_shift) < c.max_pages && entry >= 0 && entry < c.n_pages ? entry : -1;
    }
    __device__ __forceinline__ int k_page(const FmKv &c, int pos0) const { return checked(c, k, pos0 + 16 * ((threadIdx.x & 15) >> 2)); }
    __device__ __forceinline__ int v_page(const FmKv &c, int pos0) const { return checked(c, v, pos0 + 16 * ((threadIdx.x & 63) >> 4)); }
};

// A wave's columns: running maximum (of scores in units of log2), sum and output, the codes of the step
// in hand, and the step.  The queries lie in LDS as operands [piece][k step][lane], the same for the
// workgroup's waves: registers go to the codes in flight.
template <int D, int NP, bool ONCE>
struct Columns {
    static constexpr int KS = D / 32, DT = D / 16;
    fm_v4f o[DT];
    float m, l;
    int qpow, ref;           // 2^qpow takes a score back from the power of two in q; o is held in units of 2^ref
    fm_v4u kc[D / 64][4], vc[DT];
    float ks, vs;

    // (codes that nobody else reads are not kept in the caches)
    static __device__ __forceinline__ fm_v4u ld(const int8_t *p) {
        if constexpr (ONCE) return __builtin_nontemporal_load((const fm_v4u *)p);
        else return *(const fm_v4u *)p;
    }

    // Lane 16 g + column: dims 64 c + 16 g + 8 hh + j are element j of k step 2 c + hh.  Each wave fetches and
    // writes a quarter of the k steps (D 64: the first two waves a half); the columns' largest elements meet in LDS.
    // (A column that is not there holds the first row's: nothing of it is used.)
    static constexpr int MY = (KS + 3) / 4;
    fm_v4f x[MY][2];
    template <bool BF16>
    __device__ __forceinline__ void fetch_q(const void *base, int64_t at) {
        const int g = (threadIdx.x & 63) >> 4, wave = threadIdx.x >> 6;
#pragma unroll
        for (int u = 0; u < MY; u++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int s = min(wave * MY + u, KS - 1);
                x[u][h] = fm_ld4<BF16>(base, at + 64 * (s >> 1) + 16 * g + 8 * (s & 1) + 4 * h);
            }
    }
    __device__ __forceinline__ void put_q(int wave, fm_v8h *q, float (*s_big)[16]) {
        const int lane = threadIdx.x & 63, col = lane & 15;
        float big = 0.0f;
#pragma unroll
        for (int u = 0; u < MY; u++)
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++) big = fmaxf(big, fabsf(x[u][h][i]));
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        if (lane < 16) s_big[wave][col] = big;
        lds_barrier();
        big = fmaxf(fmaxf(s_big[0][col], s_big[1][col]), fmaxf(s_big[2][col], s_big[3][col]));
        qpow = q_power(big);
        const float up = power2(-qpow);
#pragma unroll
        for (int u = 0; u < MY; u++) {
            fm_v8h v[NP];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                _Float16 piece[NP];
                split<NP>(x[u][j >> 2][j & 3] * up, piece);
#pragma unroll
                for (int p = 0; p < NP; p++) v[p][j] = piece[p];
            }
            const int s = min(wave * MY + u, KS - 1);
#pragma unroll
            for (int p = 0; p < NP; p++) q[(p * KS + s) * 64 + lane] = v[p];
        }
        m = -INFINITY;
        l = 0.0f;
        ref = NO_REF;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = fm_v4f{0.f, 0.f, 0.f, 0.f};
    }

    // (a page that is not there is read as page 0 and masked)
    __device__ __forceinline__ const int8_t *k_base(const FmKv &c, const Runs &p, int h, int pos0) const {
        const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
        return c.k + fm_kv_k_at(c, D, max(p.k_page(c, pos0), 0), h, pos0 + 16 * (r >> 2) + (r & 3), 16 * g);
    }
    __device__ __forceinline__ const int8_t *v_base(const FmKv &c, const Runs &p, int h, int pos0) const {
        const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
        return c.v + fm_kv_v_at(c, D, max(p.v_page(c, pos0), 0), h, pos0 + 16 * g, r);
    }
    __device__ __forceinline__ void load_k(const int8_t *kb, int d, int t) { kc[d][t] = ld(kb + 4 * t * D + 64 * d); }
    __device__ __forceinline__ void load_v(const FmKv &c, const int8_t *vb, int d) { vc[d] = ld(vb + 16 * d * c.page_tokens); }
    __device__ __forceinline__ void load_scales(const FmKv &c, const Runs &p, int h, int pos0) {
        const int64_t at = (int64_t)max(p.v_page(c, pos0), 0) * c.kv_heads + h;
        ks = c.k_scale[at];
        vs = c.v_scale[at];
    }
    __device__ __forceinline__ void first(const FmKv &c, const Runs &p, int h, int pos0, bool any) {
        if (!any) return;
        const int8_t *kb = k_base(c, p, h, pos0), *vb = v_base(c, p, h, pos0);
#pragma unroll
        for (int d = 0; d < D / 64; d++)
#pragma unroll
            for (int t = 0; t < 4; t++) load_k(kb, d, t);
        load_scales(c, p, h, pos0);
#pragma unroll
        for (int d = 0; d < DT; d++) load_v(c, vb, d);
    }

    // 64 keys from position pos0, in the pages `now`; the column sees keys below `limit`.  MORE: each code register
    // takes the next step's (positions pos1, pages `next`) as soon as it is used.
    template <bool MORE>
    __device__ __forceinline__ void step(const FmKv &c, float scale_log2, int h, int pos0, int limit, const Runs &now, int pos1, const Runs &next,
                                         const fm_v8h *q) {
        const int g = (threadIdx.x & 63) >> 4;
        const int vpos = pos0 + 16 * g;
        const int8_t *kb = k_base(c, next, h, pos1), *vb = v_base(c, next, h, pos1);
        fm_v4f sc[4];
#pragma unroll
        for (int t = 0; t < 4; t++) sc[t] = fm_v4f{0.f, 0.f, 0.f, 0.f};
        // (the scheduler may not move loads ahead of the uses whose registers they take: it would need both)
#pragma unroll
        for (int d = 0; d < D / 64; d++) {
            fm_v8h b0[NP], b1[NP];
#pragma unroll
            for (int p = 0; p < NP; p++) b0[p] = q[(p * KS + 2 * d) * 64], b1[p] = q[(p * KS + 2 * d + 1) * 64];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const fm_v8h a0 = codes_f16(kc[d][t][0], kc[d][t][1]), a1 = codes_f16(kc[d][t][2], kc[d][t][3]);
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    sc[t] = mfma(a0, b0[p], sc[t]);
                    sc[t] = mfma(a1, b1[p], sc[t]);
                }
            }
            if constexpr (MORE) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < 4; t++) load_k(kb, d, t);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        // (scales behind the last key may be anything)
        const bool live = now.v_page(c, pos0) >= 0 && vpos < limit;
        const float f = ldexpf((live ? ks : 0.0f) * scale_log2, qpow);
        float v_scale = live ? vs : 0.0f;
        if constexpr (MORE) load_scales(c, next, h, pos1);
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sc[t][i] = live && vpos + 4 * t + i < limit ? sc[t][i] * f : -INFINITY;
                top = fmaxf(top, sc[t][i]);
            }
        const float m1 = fmaxf(m, column_max(top));
        // (nothing seen yet: any finite base keeps e^(-inf - base) at 0)
        const float base = m1 == -INFINITY ? 0.0f : m1;
        const float keep = fast_exp2(m - base);
        const int left = ref_falls(ref, m, base);
        m = m1;
        l *= keep;
        const int up = column_max(max(left, ref_of(v_scale, top, base)));
        const float keep_o = ldexpf(keep, ref - up);
        ref = up;
        v_scale = ldexpf(v_scale, -up);
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= keep_o;
        fm_v8h p8[WP][2];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e = weight(sc[t][i], base);
                l += e;
                _Float16 piece[WP];
                split<WP>(e * v_scale, piece);
                const int j = 4 * (t & 1) + i;
#pragma unroll
                for (int p = 0; p < WP; p++) p8[p][t >> 1][j] = piece[p];
            }
#pragma unroll
        for (int d0 = 0; d0 < DT; d0 += 4) {
#pragma unroll
            for (int d = d0; d < d0 + 4; d++) {
                const fm_v8h a0 = codes_f16(vc[d][0], vc[d][1]), a1 = codes_f16(vc[d][2], vc[d][3]);
#pragma unroll
                for (int p = 0; p < WP; p++) {
                    o[d] = mfma(a0, p8[p][0], o[d]);
                    o[d] = mfma(a1, p8[p][1], o[d]);
                }
            }
            if constexpr (MORE) {
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = d0; d < d0 + 4; d++) load_v(c, vb, d);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
};

// The steps of all sequences, heads and tiles are numbered through and shared out evenly: sequences
// of a batch differ in length by any factor, and only the device knows the lengths.  Every workgroup adds
// them up itself.  first[s]: steps before sequence s.  256 threads.
struct Shares {
    int first[FM_MAX_SEQ + 1], len[FM_MAX_SEQ];
    int of_wave[4];
};
__device__ __forceinline__ void add_steps(const FmKv &c, const FmAttn &a, const FmSeqs &b, Shares &sh) {
    const int t = threadIdx.x, lane = t & 63;
    int n = 0;
    if (t < b.n_seq) {
        const int len = c.len[t];
        sh.len[t] = len;
        n = c.kv_heads * fm_attn_head_steps(fm_seq_rows(b, t), a.group, a.wide, a.narrow_most, len, a.max_len);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(n, o);
        if (lane >= o) n += up;
    }
    if (lane == 63) sh.of_wave[t >> 6] = n;
    __syncthreads();
    for (int w = 0; w < t >> 6; w++) n += sh.of_wave[w];
    if (t < b.n_seq) sh.first[t + 1] = n;
    if (t == 0) sh.first[0] = 0;
    __syncthreads();
}

// Narrow tiles: a workgroup takes its share of the steps, tile by tile; the four waves take a tile's steps
// in turn and are joined through LDS.
// Bound by the codes' way from memory: 32 sequences of 8300 tokens on average, 2 cache heads of 256 in bf16, 272 MB
// in 68 us, 4.0 TB/s; one sequence of 999 by latency, 12.5 us (lengths, table, codes, join wait for each other) and
// 4 us for the join of the parts.
template <int D, bool BF16, bool ONCE>
__global__ __launch_bounds__(256, fm_attn_per_cu(D)) void fm_attn_narrow(FmKv c, FmAttn a, FmSeqs b) {
    constexpr int NP = BF16 ? 1 : 2, DT = D / 16;
    __shared__ float s_o[3][DT][64][4];
    __shared__ float s_big[4][16], s_m[4][16], s_l[4][16];   // (wave 0 may still read s_m when the others take the next tile)
    __shared__ int s_ref[4][16];
    __shared__ fm_v8h s_q[NP * (D / 32) * 64];
    __shared__ Shares sh;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    add_steps(c, a, b, sh);
    const int total = sh.first[b.n_seq], share = fm_attn_share(total, a.groups);
    if (blockIdx.x == 0)                                         // for the join
        for (int i = threadIdx.x; i <= b.n_seq; i += 256) a.first[i] = sh.first[i];
    int at = blockIdx.x * share;
    const int stop = min(total, at + share);
    if (at >= stop) return;
    int s = 0;
    for (int hi = b.n_seq; hi - s > 1;) {
        const int mid = (s + hi) / 2;
        if (sh.first[mid] <= at) s = mid;
        else hi = mid;
    }
    while (at < stop) {
        while (sh.first[s + 1] <= at) s++;                       // (sequences without rows have no steps)
        const int n = fm_seq_rows(b, s), len = __builtin_amdgcn_readfirstlane(sh.len[s]), per_head = (sh.first[s + 1] - sh.first[s]) / c.kv_heads;
        const int h = (at - sh.first[s]) / per_head;
        int off = (at - sh.first[s]) - h * per_head, tile = 0, steps;
        while (off >= (steps = fm_attn_steps(n, a.group, a.wide, len, a.max_len, tile))) off -= steps, tile++;
        const int s0 = off, s1 = min(steps, off + stop - at);    // this workgroup's steps of the tile
        at += s1 - s0;

        const int n_cols = n * a.group, cc = tile * COLS + col;
        const bool there = cc < n_cols;
        const int i = there ? cc / a.group : 0, qh = h * a.group + (there ? cc % a.group : 0);
        const int limit = there ? min(min(len, a.max_len), len - n + i + 1) : 0;
        const int64_t row = fm_seq_row0(b, s) + i;
        const int32_t *table = c.pages + (int64_t)s * c.max_pages;
        Columns<D, NP, ONCE> w;
        Runs now, next;
        int pos = (s0 + wave) * BK;
        const int end = s1 * BK;
        const bool any = pos < end;
        now.load(c, table, any ? pos : 0);
        next.load(c, table, pos + 4 * BK < end ? pos + 4 * BK : 0);
        // (the queries first: who looks at a load's result waits for all that were issued before it)
        w.template fetch_q<BF16>(a.q, row * a.q_stride + (int64_t)qh * D);
        w.first(c, now, h, any ? pos : 0, any);
        w.put_q(wave, s_q, s_big);
        lds_barrier();
        const fm_v8h *q = s_q + lane;
        if (any) {
            for (; pos + 4 * BK < end; pos += 4 * BK) {
                Runs later;
                later.load(c, table, min(pos + 8 * BK, end - BK));
                w.template step<true>(c, a.scale_log2, h, pos, limit, now, pos + 4 * BK, next, q);
                now = next;
                next = later;
            }
            w.template step<false>(c, a.scale_log2, h, pos, limit, now, pos, now, q);
        }
        w.l += __shfl_xor(w.l, 16);
        w.l += __shfl_xor(w.l, 32);

        // join the waves: wave 0 takes the others' sums at the common maximum and power of two
        __syncthreads();                                          // (the last tile's sums have been read)
        if (g == 0) s_m[wave][col] = w.m, s_l[wave][col] = w.l, s_ref[wave][col] = w.ref;
        __syncthreads();
        const float m = fmaxf(fmaxf(s_m[0][col], s_m[1][col]), fmaxf(s_m[2][col], s_m[3][col]));
        const float base = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
        int ref = NO_REF;
#pragma unroll
        for (int v = 0; v < 4; v++) {
            l = fmaf(s_l[v][col], fast_exp2(s_m[v][col] - base), l);
            ref = max(ref, ref_falls(s_ref[v][col], s_m[v][col], base));
        }
        // (a part of a tile is normalised as well: its output is a mean of values; the power of two before the sum, or a
        // small weight of large values would fall below fp32 in between)
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const float f = ldexpf(fast_exp2(w.m - base), w.ref - ref) * inv;
#pragma unroll
        for (int d = 0; d < DT; d++) w.o[d] *= f;
        if (wave) {
#pragma unroll
            for (int d = 0; d < DT; d++) *(fm_v4f *)s_o[wave - 1][d][lane] = w.o[d];
        }
        __syncthreads();
        if (wave) continue;
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int v = 0; v < 3; v++) w.o[d] += *(const fm_v4f *)s_o[v][d][lane];
        // register i of tile d: dim 16 d + 4 g + i
#pragma unroll
        for (int d = 0; d < DT; d++) w.o[d] = times_power2(w.o[d], ref);
        if (s0 == 0 && s1 == steps) {
            if (!there) continue;
            const int64_t to = (row * a.q_heads + qh) * D + 4 * g;
#pragma unroll
            for (int d = 0; d < DT; d++) fm_st4<BF16>(a.out, to + 16 * d, w.o[d]);
        } else {
            const int64_t to = (int64_t)fm_attn_slot(blockIdx.x, s0) * COLS + col;
#pragma unroll
            for (int d = 0; d < DT; d++) *(fm_v4f *)(a.part_o + to * D + 16 * d + 4 * g) = w.o[d];
            if (g == 0) a.part_ml[2 * to] = m, a.part_ml[2 * to + 1] = l;
        }
    }
}

// Wide tiles: 128 columns of one (sequence, cache head), 64 with two pieces.  The workgroup turns a step's codes
// into fp16 operands in LDS once, [tile][k step][lane] of 16 bytes; the queries lie there too.  Eight waves:
// wave w has the columns of group w & 3 (16 CT of them) and one half of a step's keys, w >> 2, with a
// running maximum, sum and output of its own; the halves are joined at the tile's end.  Two waves per
// SIMD, so that one's softmax runs beside the other's products, in 256 registers each.
// The codes of the next step are on their way in registers meanwhile; keys are replaced behind the first
// product's barrier, values behind the second's, so a step has two barriers and one copy of each.
// 2048 rows over 8192 keys, 16 heads of 256, bf16: 241 GFLOP in 403 us, 598 TFLOP/s (a large library product 1050);
// with one piece of p and a power of two that goes by the value scales alone 326 us.  A step of 128 columns x 64 keys x
// 256 dims has products for 3072 cycles a SIMD (1024 of the scores, 2048 of the two pieces), 41 % of its time; the vector
// ALU is busy for 61 %, with two waves per SIMD and two barriers.  Heads of 256 in bf16 spill 2 registers.
template <int D, bool BF16>
__global__ __launch_bounds__(512, 2) void fm_attn_wide(FmKv c, FmAttn a, FmSeqs b, FmWide w) {
    constexpr int NP = BF16 ? 1 : 2, CT = BF16 ? 2 : 1, KS = D / 32, DT = D / 16, LD = D / 64, WIDE = 64 * CT;
    constexpr int UNITS = 4 * LD, MY = (UNITS + 7) / 8;          // loads of a wave and step, for K and for V
    // K [4][KS][64] | V [DT][2][64] | q [4][CT][NP][KS][64], then o of four waves [4][CT][DT][64]
    constexpr int K_AT = 0, V_AT = 4 * KS * 64, Q_AT = V_AT + DT * 2 * 64, ALL = Q_AT + 4 * CT * NP * KS * 64;
    constexpr int O_ALL = 4 * CT * DT * 64;
    __shared__ fm_v8h lds[ALL > O_ALL ? ALL : O_ALL];
    __shared__ float s_m[4][CT][16], s_l[4][CT][16];
    __shared__ int s_ref[4][CT][16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const int cg = wave & 3, half = wave >> 2;
    const fm_v8h *s_k = lds + K_AT + lane, *s_v = lds + V_AT + lane;
    fm_v8h *s_q = lds + Q_AT + cg * CT * NP * KS * 64 + lane;
    const int units = w.first[b.n_seq] * c.kv_heads * a.splits;
    for (int round = 0; round * a.groups < units; round++) {
        const int unit = fm_attn_wide_pick(round, blockIdx.x, a.groups);
        if (unit >= units) continue;
        const FmWideUnit at = fm_attn_wide_unit(w, b.n_seq, c.kv_heads, a.splits, unit);
        const int s = at.s, h = at.h, tile = at.tile, n = fm_seq_rows(b, s), len = __builtin_amdgcn_readfirstlane(c.len[s]);
        const int steps = fm_attn_steps(n, a.group, WIDE, len, a.max_len, tile);
        const int s0 = (int)((int64_t)steps * at.part / a.splits), s1 = (int)((int64_t)steps * (at.part + 1) / a.splits);
        const int32_t *table = c.pages + (int64_t)s * c.max_pages;
        Runs now, next;
        now.load(c, table, s0 * BK);
        next.load(c, table, max(min(s0 + 1, s1 - 1), 0) * BK);
        fm_v4f o[CT][DT];
        float m[CT], l[CT];
        int qpow[CT], ref[CT], limit[CT], all_limit = 0x7FFFFFFF;
        int64_t to[CT];          // the column's place in the output, -1 if it is not there
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            const int cc = tile * WIDE + (cg * CT + ct) * 16 + r;
            const bool there = cc < n * a.group;
            const int i = there ? cc / a.group : 0, qh = h * a.group + (there ? cc % a.group : 0);
            const int64_t row = fm_seq_row0(b, s) + i;
            limit[ct] = there ? min(min(len, a.max_len), len - n + i + 1) : 0;
            all_limit = min(all_limit, limit[ct]);
            to[ct] = there ? (row * a.q_heads + qh) * D : -1;
            fm_v4f x[KS][2];
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int hh = 0; hh < 2; hh++)
                    x[k][hh] = fm_ld4<BF16>(a.q, row * a.q_stride + (int64_t)qh * D + 64 * (k >> 1) + 16 * g + 8 * (k & 1) + 4 * hh);
            float big = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++)
#pragma unroll
                for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(x[k][j >> 2][j & 3]));
            big = fmaxf(big, __shfl_xor(big, 16));
            big = fmaxf(big, __shfl_xor(big, 32));
            qpow[ct] = q_power(big);
            const float up = power2(-qpow[ct]);
            // (both halves' waves have the columns: each writes half of the k steps)
            if (!ct) lds_barrier();                               // (the last tile's operands have been read)
#pragma unroll
            for (int k = 0; k < KS; k++) {
                if ((k & 1) != half) continue;
                fm_v8h v[NP];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    _Float16 piece[NP];
                    split<NP>(x[k][j >> 2][j & 3] * up, piece);
#pragma unroll
                    for (int p = 0; p < NP; p++) v[p][j] = piece[p];
                }
#pragma unroll
                for (int p = 0; p < NP; p++) s_q[((ct * NP + p) * KS + k) * 64] = v[p];
            }
            m[ct] = -INFINITY;
            l[ct] = 0.0f;
            ref[ct] = NO_REF;
#pragma unroll
            for (int d = 0; d < DT; d++) o[ct][d] = fm_v4f{0.f, 0.f, 0.f, 0.f};
        }
        for (int x = 32; x; x >>= 1) all_limit = min(all_limit, __shfl_xor(all_limit, x));
        // this wave's loads: unit u of K is tile u & 3, dims 64 (u >> 2) ..; of V dims 16 u ..
        fm_v4u kc[MY], vc[MY];
        float ks, vs;
        auto fetch = [&](const Runs &p, int pos) {
            const int64_t sc = (int64_t)max(p.v_page(c, pos), 0) * c.kv_heads + h;
            const int8_t *kb = c.k + fm_kv_k_at(c, D, max(p.k_page(c, pos), 0), h, pos + 16 * (r >> 2) + (r & 3) + 4 * (wave & 3), 16 * g);
            const int8_t *vb = c.v + fm_kv_v_at(c, D, max(p.v_page(c, pos), 0), h, pos + 16 * g, r);
#pragma unroll
            for (int j = 0; j < MY; j++) kc[j] = *(const fm_v4u *)(kb + 64 * (min(wave + 8 * j, UNITS - 1) >> 2));
#pragma unroll
            for (int j = 0; j < MY; j++) vc[j] = *(const fm_v4u *)(vb + 16 * min(wave + 8 * j, UNITS - 1) * c.page_tokens);
            ks = c.k_scale[sc];
            vs = c.v_scale[sc];
        };
        auto put_k = [&]() {
#pragma unroll
            for (int j = 0; j < MY; j++) {
                const int u = wave + 8 * j;
                if (u >= UNITS) continue;
                fm_v8h *z = lds + K_AT + ((u & 3) * KS + 2 * (u >> 2)) * 64 + lane;
                z[0] = codes_f16(kc[j][0], kc[j][1]);
                z[64] = codes_f16(kc[j][2], kc[j][3]);
            }
        };
        auto put_v = [&]() {
#pragma unroll
            for (int j = 0; j < MY; j++) {
                const int u = wave + 8 * j;
                if (u >= UNITS) continue;
                fm_v8h *z = lds + V_AT + u * 128 + lane;
                z[0] = codes_f16(vc[j][0], vc[j][1]);
                z[64] = codes_f16(vc[j][2], vc[j][3]);
            }
        };
        fetch(now, s0 * BK);
        put_k();
        for (int st = s0; st < s1; st++) {
            const int pos = st * BK, vpos = pos + 16 * g + 8 * half;      // first of this lane's eight keys
            const float k_scale = ks * a.scale_log2, v_scale0 = vs;
            const bool there = now.v_page(c, pos) >= 0;
            lds_barrier();                                        // the step's keys are there, the last one's values read
            put_v();
            Runs later;
            later.load(c, table, min(st + 2, s1 - 1) * BK);
            fetch(next, min(st + 1, s1 - 1) * BK);
            fm_v4f sc[CT][2];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) sc[ct][0] = sc[ct][1] = fm_v4f{0.f, 0.f, 0.f, 0.f};
            // operands are read a group of products ahead (the scheduler would put each read in front of its use)
            fm_v8h xk[2][2], yq[2][CT * NP];
            auto read_k = [&](int k) {
                xk[k & 1][0] = s_k[(2 * half * KS + k) * 64];
                xk[k & 1][1] = s_k[((2 * half + 1) * KS + k) * 64];
#pragma unroll
                for (int y = 0; y < CT * NP; y++) yq[k & 1][y] = s_q[(y * KS + k) * 64];
            };
            read_k(0);
#pragma unroll
            for (int k = 0; k < KS; k++) {
                if (k + 1 < KS) read_k(k + 1);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int p = 0; p < NP; p++) {
                        sc[ct][0] = mfma(xk[k & 1][0], yq[k & 1][ct * NP + p], sc[ct][0]);
                        sc[ct][1] = mfma(xk[k & 1][1], yq[k & 1][ct * NP + p], sc[ct][1]);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
            lds_barrier();                                        // the keys have been read, the values are there
            fm_v8h xv[2][2];
            auto read_v = [&](int d0) {
#pragma unroll
                for (int d = 0; d < 2; d++) xv[d0 >> 1 & 1][d] = s_v[((d0 + d) * 2 + half) * 64];
            };
            read_v(0);
            if (st + 1 < s1) put_k();
            const bool whole = __all(there) && pos + BK <= all_limit;      // nothing of the step is masked
            fm_v8h p8[CT][WP];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const bool live = there && vpos < limit[ct];
                const float f = ldexpf(live ? k_scale : 0.0f, qpow[ct]);
                float v_scale = live ? v_scale0 : 0.0f, top = -INFINITY;
                if (whole) {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[ct][t][i] *= f, top = fmaxf(top, sc[ct][t][i]);
                } else {
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            sc[ct][t][i] = live && vpos + 4 * t + i < limit[ct] ? sc[ct][t][i] * f : -INFINITY;
                            top = fmaxf(top, sc[ct][t][i]);
                        }
                }
                const float m1 = fmaxf(m[ct], column_max(top)), base = m1 == -INFINITY ? 0.0f : m1;
                const float keep = fast_exp2(m[ct] - base);
                const int left = ref_falls(ref[ct], m[ct], base);
                m[ct] = m1;
                const int up = column_max(max(left, ref_of(v_scale, top, base)));
                const float keep_o = ldexpf(keep, ref[ct] - up);
                ref[ct] = up;
                v_scale = ldexpf(v_scale, -up);
                l[ct] *= keep;
                if (!__all(keep_o == 1.0f)) {
#pragma unroll
                    for (int d = 0; d < DT; d++) o[ct][d] *= keep_o;
                }
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float e = weight(sc[ct][t][i], base);
                        l[ct] += e;
                        _Float16 piece[WP];
                        split<WP>(e * v_scale, piece);
#pragma unroll
                        for (int p = 0; p < WP; p++) p8[ct][p][4 * t + i] = piece[p];
                    }
            }
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += 2) {
                if (d0 + 2 < DT) read_v(d0 + 2);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int d = 0; d < 2; d++)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++)
#pragma unroll
                        for (int p = 0; p < WP; p++) o[ct][d0 + d] = mfma(xv[d0 >> 1 & 1][d], p8[ct][p], o[ct][d0 + d]);
                __builtin_amdgcn_sched_barrier(0);
            }
            now = next;
            next = later;
        }
        // the second halves' outputs to the first halves' waves, at the common maximum and power of two
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            l[ct] += __shfl_xor(l[ct], 16);
            l[ct] += __shfl_xor(l[ct], 32);
        }
        lds_barrier();                                            // operands have been read
        if (half) {
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                if (g == 0) s_m[cg][ct][r] = m[ct], s_l[cg][ct][r] = l[ct], s_ref[cg][ct][r] = ref[ct];
#pragma unroll
                for (int d = 0; d < DT; d++) *(fm_v4f *)(lds + ((cg * CT + ct) * DT + d) * 64 + lane) = o[ct][d];
            }
        }
        lds_barrier();
        if (half) continue;
#pragma unroll
        for (int ct = 0; ct < CT; ct++) {
            if (to[ct] < 0) continue;
            const float m2 = s_m[cg][ct][r], both = fmaxf(m[ct], m2), base = both == -INFINITY ? 0.0f : both;
            const float e1 = fast_exp2(m[ct] - base), e2 = fast_exp2(m2 - base);
            const int ref2 = s_ref[cg][ct][r], top = max(ref_falls(ref[ct], m[ct], base), ref_falls(ref2, m2, base));
            const float sum = e1 * l[ct] + e2 * s_l[cg][ct][r];
            // (a part of a tile is normalised as well: its output is a mean of values)
            const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
            const float f1 = ldexpf(e1, ref[ct] - top) * inv, f2 = ldexpf(e2, ref2 - top) * inv;
            const int64_t part = (int64_t)unit * WIDE + (cg * CT + ct) * 16 + r;
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const fm_v4f z = times_power2(o[ct][d] * f1 + *(const fm_v4f *)(lds + ((cg * CT + ct) * DT + d) * 64 + lane) * f2, top);
                if (a.splits == 1) fm_st4<BF16>(a.out, to[ct] + 16 * d + 4 * g, z);
                else *(fm_v4f *)(a.part_o + part * D + 16 * d + 4 * g) = z;
            }
            if (a.splits > 1 && g == 0) a.part_ml[2 * part] = both, a.part_ml[2 * part + 1] = sum;
        }
    }
}

// One column out of `parts` parts, by a wave: D / 64 dims a lane, a lane per part for its weight, its sum at
// the common maximum over all of them.  slot(k): where part k's column lies.
template <int D, bool BF16, class Slot>
__device__ __forceinline__ void join_column(const FmAttn &a, int parts, Slot slot, int64_t to) {
    const int lane = threadIdx.x & 63;
    auto of = [&](int k) { return k < parts ? *(const float2 *)(a.part_ml + 2 * slot(k)) : float2{-INFINITY, 0.0f}; };
    const float2 first = of(lane);
    float m = first.x;
    for (int k = lane + 64; k < parts; k += 64) m = fmaxf(m, of(k).x);
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float base = m == -INFINITY ? 0.0f : m, first_l = fast_exp2(first.x - base) * first.y;
    float l = first_l, o[D / 64];
    for (int k = lane + 64; k < parts; k += 64) {
        const float2 p = of(k);
        l = fmaf(fast_exp2(p.x - base), p.y, l);
    }
    l = fm_group_sum<64>(l);
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
    for (int d = 0; d < D / 64; d++) o[d] = 0.0f;
    for (int k0 = 0; k0 < parts; k0 += 64) {
        const int some = min(64, parts - k0);
        float f = first_l;
        if (k0) {
            const float2 p = of(k0 + lane);
            f = fast_exp2(p.x - base) * p.y;
        }
        f *= inv;
#pragma unroll 4
        for (int k = 0; k < some; k++) {
            const float *p = a.part_o + slot(k0 + k) * D + lane;
            const float fk = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), k));
#pragma unroll
            for (int d = 0; d < D / 64; d++) o[d] = fmaf(fk, p[64 * d], o[d]);
        }
    }
#pragma unroll
    for (int d = 0; d < D / 64; d++) fm_st1<BF16>(a.out, to + 64 * d + lane, o[d]);
}

// Narrow tiles that several workgroups took: four columns a workgroup.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void fm_attn_join(FmKv c, FmAttn a, FmSeqs b) {
    const int s = blockIdx.z, h = blockIdx.y, tile = blockIdx.x >> 2;
    const int n = fm_seq_rows(b, s);
    if (tile >= fm_attn_tiles(n, a.group, 0, a.narrow_most)) return;
    const int len = c.len[s], from = a.first[s], per_head = (a.first[s + 1] - from) / c.kv_heads;
    const int share = fm_attn_share(a.first[b.n_seq], a.groups), steps = fm_attn_steps(n, a.group, 0, len, a.max_len, tile);
    int at = from + h * per_head;
    for (int t = 0; t < tile; t++) at += fm_attn_steps(n, a.group, 0, len, a.max_len, t);
    const int g0 = at / share, g1 = (at + steps - 1) / share;
    if (g0 == g1) return;
    const int col = 4 * (blockIdx.x & 3) + (threadIdx.x >> 6), cc = tile * COLS + col;
    if (cc >= n * a.group) return;
    join_column<D, BF16>(a, g1 - g0 + 1, [&](int k) { return (int64_t)fm_attn_slot(g0 + k, (g0 + k) * share - at) * COLS + col; },
                         ((int64_t)(fm_seq_row0(b, s) + cc / a.group) * a.q_heads + h * a.group + cc % a.group) * D);
}

// Wide tiles in parts: four columns a workgroup.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void fm_attn_wide_join(FmKv c, FmAttn a, FmSeqs b, FmWide w) {
    const int tile = blockIdx.x / (a.wide / 4), col = 4 * (blockIdx.x % (a.wide / 4)) + (threadIdx.x >> 6);
    const FmWideUnit at = fm_attn_wide_unit(w, b.n_seq, c.kv_heads, a.splits, tile * a.splits);
    const int cc = at.tile * a.wide + col;
    if (cc >= fm_seq_rows(b, at.s) * a.group) return;
    join_column<D, BF16>(a, a.splits, [&](int k) { return ((int64_t)tile * a.splits + k) * a.wide + col; },
                         ((int64_t)(fm_seq_row0(b, at.s) + cc / a.group) * a.q_heads + at.h * a.group + cc % a.group) * D);
}

// ---- the cache's rows --------------------------------------------------------------------------
// code = value / scale rounded to nearest even, decided as in real numbers: fp32 operands have 24
// bits, so a quotient that is not half-way between two codes is further than 2^-33 from there, and
// the fp64 quotient (2^-53) falls on the same side.
__device__ __forceinline__ int quantise(double x, float scale) {
    if (x != x) return 0;
    if (!(scale > 0.0f)) return x > 1.7e308 ? 127 : x < -1.7e308 ? -127 : 0;
    const double q = rint(x / (double)scale);
    return q > 127.0 ? 127 : q < -127.0 ? -127 : (int)q;
}

// The same decision in fp32, for a scale well inside the range: the candidate from x * (1 / scale) is off by
// at most one code, and the sign of x - (code +- 1/2) scale, one fma, tells (an fma's sign is that of the
// exact value while nothing underflows).
__device__ __forceinline__ int quantise_fast(float x, float scale, float inv) {
    float c = rintf(x * inv);
    const float up = fmaf(-(c + 0.5f), scale, x), down = fmaf(-(c - 0.5f), scale, x);
    const bool odd = (int)c & 1;
    if (up > 0.0f || (up == 0.0f && odd)) c += 1.0f;
    else if (down < 0.0f || (down == 0.0f && odd)) c -= 1.0f;
    c = fminf(fmaxf(c, -127.0f), 127.0f);
    return fabsf(x) < INFINITY ? (int)c : x > 0.0f ? 127 : x < 0.0f ? -127 : 0;
}

constexpr int KV_T = 1024, KV_E = 128 * 256 / 4 / KV_T;    // threads; float4 a thread of the largest page

// One workgroup: the rows that fall into one page of one sequence, for one head, keys (z even) or
// values.  The rows are read once, into registers: their largest magnitude, then the codes.  Values
// are turned through LDS, so that both the rows and the page move in whole lines: a page that gets a
// run of tokens is rewritten (its other bytes as they are); fewer than 16 tokens go byte by byte.  (With the read
// back, rewritten / byte by byte: one sequence 8 rows 10.2 / 9.7 us, 16 rows 10.9 / 10.6, 32 rows 11.4 / 12.4; 32
// sequences 4 rows 10.6 / 10.5, 16 rows 11.5 / 13.7.)  Bound by latency: 1500 rows of 2 heads of 256 take 10 us.
template <bool BF16>
__global__ __launch_bounds__(KV_T) void fm_kv_append(FmKv c, FmKvRows x, int D, FmSeqs b) {
    __shared__ float red[KV_T / 64];
    __shared__ __attribute__((aligned(16))) int8_t turn[256 * (128 + 4)];   // [dim][token], rows a bank apart
    const int s = blockIdx.z >> 1, h = blockIdx.y, tid = threadIdx.x;
    const bool value = blockIdx.z & 1;
    const int P = c.page_tokens, ps = c.page_shift, LD = P + 4, s4 = 31 - __builtin_clz(D) - 2, d4 = 1 << s4;
    FmKvSpan sp;
    if (!fm_kv_span(fm_seq_rows(b, s), c.len[s], c.page_shift, blockIdx.x, &sp)) return;
    const int page = fm_kv_page(c, s, sp.start);
    if (page < 0) return;
    const int t0 = sp.t0, n = sp.t1 - sp.t0;                          // tokens written, in the page
    const int64_t row0 = (int64_t)fm_seq_row0(b, s) + sp.row0 + t0;  // the first one's row
    const void *src = value ? x.v : x.k;
    const int64_t stride = value ? x.v_stride : x.k_stride;
    float *scale_at = (value ? c.v_scale : c.k_scale) + (int64_t)page * c.kv_heads + h;
    const float old = t0 > 0 ? *scale_at : 0.0f;
    fm_v4f w[KV_E];
    float big = 0.0f;
#pragma unroll
    for (int u = 0; u < KV_E; u++) {
        const int e = tid + u * KV_T;
        if (e < n * d4) w[u] = fm_ld4<BF16>(src, (row0 + (e >> s4)) * stride + (int64_t)h * D + 4 * (e & (d4 - 1)));
    }
#pragma unroll
    for (int u = 0; u < KV_E; u++)
        if (tid + u * KV_T < n * d4)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float m = fabsf(w[u][i]);
                if (m < INFINITY) big = fmaxf(big, m);
            }
    for (int o = 32; o; o >>= 1) big = fmaxf(big, __shfl_xor(big, o));
    if ((tid & 63) == 0) red[tid >> 6] = big;
    __syncthreads();                                             // (everybody has read the old scale, too)
#pragma unroll
    for (int i = 0; i < KV_T / 64; i++) big = fmaxf(big, red[i]);
    const float scale = fmaxf(old, big * (1.0f / 127.0f));      // (the scale is this product, not the quotient: up to an ulp apart)
    if (tid == 0) *scale_at = scale;
    int8_t *codes = value ? c.v + fm_kv_v_at(c, D, page, h, 0, 0) : c.k + fm_kv_k_at(c, D, page, h, 0, 0);
    if (t0 > 0 && scale != old) {                               // the old codes go to the new scale
        for (int e = tid; e < t0 * D; e += KV_T) {
            int8_t *at = codes + (value ? (e & (D - 1)) * P + (e >> (s4 + 2)) : e);
            *at = (int8_t)quantise((double)*at * (double)old, scale);
        }
    }
    const bool fast = scale > 0x1p-100f && scale < 0x1p100f, whole = value && n >= 16;
    const float inv = 1.0f / scale;
    if (whole) {                                                // the page as it is
        __syncthreads();
        for (int e = 4 * tid; e < P * D; e += 4 * KV_T) *(uint32_t *)(turn + (e >> ps) * LD + (e & (P - 1))) = *(const uint32_t *)(codes + e);
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < KV_E; u++) {
        const int e = tid + u * KV_T;
        if (e >= n * d4) continue;
        const int t = t0 + (e >> s4), d = 4 * (e & (d4 - 1));
        int q[4];
#pragma unroll
        for (int i = 0; i < 4; i++) q[i] = fast ? quantise_fast(w[u][i], scale, inv) : quantise((double)w[u][i], scale);
        if (value) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (whole) turn[(d + i) * LD + t] = (int8_t)q[i];
                else codes[(d + i) * P + t] = (int8_t)q[i];
            }
        } else {
            *(uint32_t *)(codes + t * D + d) = (q[0] & 255) | (q[1] & 255) << 8 | (q[2] & 255) << 16 | (uint32_t)q[3] << 24;
        }
    }
    if (whole) {
        __syncthreads();
        for (int e = 4 * tid; e < P * D; e += 4 * KV_T) *(uint32_t *)(codes + e) = *(const uint32_t *)(turn + (e >> ps) * LD + (e & (P - 1)));
    }
}

__global__ __launch_bounds__(256) void fm_kv_read(FmKv c, FmKvRows x, int D, FmSeqs b) {
    const int s = blockIdx.z, h = blockIdx.y;
    const int n = fm_seq_rows(b, s), len = c.len[s], P = c.page_tokens;
    for (int e = blockIdx.x * 256 + threadIdx.x; e < n * (D / 4); e += gridDim.x * 256) {
        const int i = e / (D / 4), d = 4 * (e % (D / 4));
        const int pos = len - n + i, page = fm_kv_page(c, s, pos);
        fm_v4f k = {0.f, 0.f, 0.f, 0.f}, v = {0.f, 0.f, 0.f, 0.f};
        if (page >= 0) {
            const int64_t ph = (int64_t)page * c.kv_heads + h;
            const float ks = c.k_scale[ph], vs = c.v_scale[ph];
            const int8_t *kc = c.k + fm_kv_k_at(c, D, page, h, pos, d), *vc = c.v + fm_kv_v_at(c, D, page, h, pos, d);
#pragma unroll
            for (int j = 0; j < 4; j++) k[j] = (float)kc[j] * ks, v[j] = (float)vc[j * P] * vs;
        }
        const int64_t row = (int64_t)fm_seq_row0(b, s) + i;
        *(fm_v4f *)(x.k_out + row * x.k_stride + (int64_t)h * D + d) = k;
        *(fm_v4f *)(x.v_out + row * x.v_stride + (int64_t)h * D + d) = v;
    }
}

template <int D, bool BF16>
void launch_attn(const FmKv &c, const FmAttn &a, const FmSeqs &b, hipStream_t st) {
    const dim3 grid(a.groups), block(256);
    if (a.wide) {
        FmWide w;
        fm_attn_wide_tiles(b, a.group, a.wide, a.narrow_most, &w);
        hipLaunchKernelGGL((fm_attn_wide<D, BF16>), grid, dim3(512), 0, st, c, a, b, w);
        if (a.splits > 1)
            hipLaunchKernelGGL((fm_attn_wide_join<D, BF16>), dim3(w.first[b.n_seq] * c.kv_heads * (a.wide / 4)), block, 0, st, c, a, b, w);
        return;
    }
    if (a.n_tiles == 1) hipLaunchKernelGGL((fm_attn_narrow<D, BF16, true>), grid, block, 0, st, c, a, b);
    else hipLaunchKernelGGL((fm_attn_narrow<D, BF16, false>), grid, block, 0, st, c, a, b);
    if (a.groups > 1) hipLaunchKernelGGL((fm_attn_join<D, BF16>), dim3(4 * a.n_tiles, c.kv_heads, b.n_seq), block, 0, st, c, a, b);
}

}  // namespace

// ws: what fm_attn_check asked for
extern "C" int fm_launch_attn(const FmKv *c, const FmAttn *args, const FmSeqs *b, int D, int bf16, void *ws, int n_cu, hipStream_t st) {
    for (int pass = 0; pass < 2; pass++) {
        const int wide = pass ? args->wide_cols : 0;
        FmAttn a = *args;
        fm_attn_plan(c, &a, b, D, n_cu, wide);
        if (!a.n_tiles) continue;
        FmWide w;
        fm_attn_wide_tiles(*b, a.group, wide, a.narrow_most, &w);
        const size_t cols = wide ? (size_t)w.first[b->n_seq] * c->kv_heads * a.splits * wide : (size_t)2 * a.groups * COLS;
        a.part_o = (float *)ws;      // (parts | maximum and sum of each | steps before each sequence)
        a.part_ml = a.part_o + cols * D;
        a.first = (int *)(a.part_ml + cols * 2);
        switch (D) {
            case 64: bf16 ? launch_attn<64, true>(*c, a, *b, st) : launch_attn<64, false>(*c, a, *b, st); break;
            case 128: bf16 ? launch_attn<128, true>(*c, a, *b, st) : launch_attn<128, false>(*c, a, *b, st); break;
            case 256: bf16 ? launch_attn<256, true>(*c, a, *b, st) : launch_attn<256, false>(*c, a, *b, st); break;
            default: return FM_ERR_UNSUPPORTED;
        }
        if (hipGetLastError() != hipSuccess) return FM_ERR_HIP;
    }
    return FM_OK;
}

extern "C" int fm_launch_kv(const FmKv *c, const FmKvRows *x, const FmSeqs *b, int D, int bf16, int read, hipStream_t st) {
    const int most = fm_most_rows(*b);
    if (most < 1) return FM_OK;
    if (read) {
        const int wg = (int)(((int64_t)most * (D / 4) + 255) / 256);
        hipLaunchKernelGGL(fm_kv_read, dim3(wg < 1024 ? wg : 1024, c->kv_heads, b->n_seq), dim3(256), 0, st, *c, *x, D, *b);
    } else {
        const dim3 grid((most + c->page_tokens - 2) / c->page_tokens + 1, c->kv_heads, 2 * b->n_seq);
        if (bf16) hipLaunchKernelGGL(fm_kv_append<true>, grid, dim3(KV_T), 0, st, *c, *x, D, *b);
        else hipLaunchKernelGGL(fm_kv_append<false>, grid, dim3(KV_T), 0, st, *c, *x, D, *b);
    }
    return hipGetLastError() == hipSuccess ? FM_OK : FM_ERR_HIP;
}
