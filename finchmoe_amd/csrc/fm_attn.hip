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
// near 2^8 (2^14 for p, whose keys' value scales ride along relative to the largest seen), far above
// the subnormals: two pieces (22 bits) for fp32 vectors, one for bf16 ones (q is then exact, p
// keeps 11 bits).
#include "fm_mix.h"

namespace {

constexpr int BK = FM_ATTN_KEYS, COLS = FM_ATTN_COLS;
constexpr float P_SHIFT = 14.0f;   // p is computed as 2^14 p

__device__ __forceinline__ fm_v4f mfma(fm_v8h a, fm_v8h b, fm_v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
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

// A wave's columns: running maximum (of scores in units of log2), sum and output, and the step that
// adds 64 keys.
template <int D, int NP>
struct Columns {
    static constexpr int KS = D / 32, DT = D / 16;
    fm_v8h q[NP][KS];
    fm_v4f o[DT];
    float m, l, qscale;      // qscale: takes a score back from the power of two in q
    int ref;                 // o is held in units of 2^ref, a power of two above every value scale seen

    // lane 16 g + column: dims 64 c + 16 g + 8 hh + j are element j of k step 2 c + hh
    template <bool BF16>
    __device__ __forceinline__ void load_q(const void *base, int64_t at, bool there, float scale_log2) {
        const int g = (threadIdx.x & 63) >> 4;
        fm_v4f x[KS][2];
        float big = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                x[s][h] = there ? fm_ld4<BF16>(base, at + 64 * (s >> 1) + 16 * g + 8 * (s & 1) + 4 * h) : fm_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 4; i++) big = fmaxf(big, fabsf(x[s][h][i]));
            }
        big = fmaxf(big, __shfl_xor(big, 16));
        big = fmaxf(big, __shfl_xor(big, 32));
        int e = (int)(__float_as_uint(big) >> 23 & 255) - 127;
        e = e > 100 ? 100 : e < -100 ? -100 : e;      // (zeros, infinities: any power will do)
        const float up = __uint_as_float((uint32_t)(127 + 8 - e) << 23);
        qscale = __uint_as_float((uint32_t)(127 - 8 + e) << 23) * scale_log2;
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float f = x[s][j >> 2][j & 3] * up;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    const _Float16 hv = (_Float16)f;
                    q[p][s][j] = hv;
                    f -= (float)hv;
                }
            }
        m = -INFINITY;
        l = 0.0f;
        ref = -100;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] = fm_v4f{0.f, 0.f, 0.f, 0.f};
    }

    // 64 keys from position pos0; the column sees keys below `limit`
    __device__ __forceinline__ void step(const FmKv &c, int s, int h, int pos0, int limit) {
        const int lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
        // keys of tile rows: run r / 4 of 16 keys; of scores and of V: run g
        const int kpos = pos0 + 16 * (r >> 2), vpos = pos0 + 16 * g;
        const int kp = fm_kv_page(c, s, kpos), vp = fm_kv_page(c, s, vpos);
        // (a page that is not there is read as page 0 and masked)
        const int8_t *kb = c.k + fm_kv_k_at(c, D, kp < 0 ? 0 : kp, h, kpos + (r & 3), 16 * g);
        const int8_t *vb = c.v + fm_kv_v_at(c, D, vp < 0 ? 0 : vp, h, vpos, r);
        const bool live = vp >= 0 && vpos < limit;
        float ks = 0.0f, vs = 0.0f;
        if (live) {
            ks = c.k_scale[(int64_t)vp * c.kv_heads + h];
            vs = c.v_scale[(int64_t)vp * c.kv_heads + h];
        }
        fm_v4f sc[4];
#pragma unroll
        for (int t = 0; t < 4; t++) sc[t] = fm_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D / 64; d++)
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const uint4 w = *(const uint4 *)(kb + 4 * t * D + 64 * d);
                const fm_v8h a0 = codes_f16(w.x, w.y), a1 = codes_f16(w.z, w.w);
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    sc[t] = mfma(a0, q[p][2 * d], sc[t]);
                    sc[t] = mfma(a1, q[p][2 * d + 1], sc[t]);
                }
            }
        const float f = ks * qscale;
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                sc[t][i] = live && vpos + 4 * t + i < limit ? sc[t][i] * f : -INFINITY;
                top = fmaxf(top, sc[t][i]);
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m1 = fmaxf(m, top);
        // (nothing seen yet: any finite base keeps e^(-inf - base) at 0)
        const float base = m1 == -INFINITY ? 0.0f : m1;
        const float keep = exp2f(m - base);
        m = m1;
        l *= keep;
        int up = live ? (int)(__float_as_uint(vs) >> 23 & 255) - 126 : -100;
        up = max(ref, min(up, 100));
        up = max(up, __shfl_xor(up, 16));
        up = max(up, __shfl_xor(up, 32));
        const float keep_o = ldexpf(keep, ref - up);
        ref = up;
        vs = ldexpf(vs, -up);
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= keep_o;
        fm_v8h p8[NP][2];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float e = exp2f(sc[t][i] - base + P_SHIFT);
                l += e;
                // (a scale behind the last key may be anything: 0 * NaN must not come in)
                float pv = e == 0.0f ? 0.0f : e * vs;
                const int j = 4 * (t & 1) + i;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    const _Float16 hv = (_Float16)pv;
                    p8[p][t >> 1][j] = hv;
                    pv -= (float)hv;
                }
            }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const uint4 w = *(const uint4 *)(vb + (int64_t)16 * d * c.page_tokens);
            const fm_v8h a0 = codes_f16(w.x, w.y), a1 = codes_f16(w.z, w.w);
#pragma unroll
            for (int p = 0; p < NP; p++) {
                o[d] = mfma(a0, p8[p][0], o[d]);
                o[d] = mfma(a1, p8[p][1], o[d]);
            }
        }
    }
};

// One workgroup: a chunk of the keys, 16 columns of one (sequence, cache head).  Its four waves take
// steps of 64 keys in turn and are joined through LDS.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void fm_attn_cols(FmKv c, FmAttn a, FmSeqs b) {
    constexpr int NP = BF16 ? 1 : 2, DT = D / 16;
    __shared__ float s_o[3][DT][64][4];
    __shared__ float s_m[4][16], s_l[4][16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, col = lane & 15;
    const int s = blockIdx.z, h = blockIdx.y, chunk = blockIdx.x % a.n_chunks, tile = blockIdx.x / a.n_chunks;
    const int n = fm_seq_rows(b, s), n_cols = n * a.group;
    if (tile * COLS >= n_cols) return;
    const int cc = tile * COLS + col;
    const bool there = cc < n_cols;
    const int i = there ? cc / a.group : 0, qh = h * a.group + (there ? cc % a.group : 0);
    const int len = c.len[s];
    const int seen = min(len, a.max_len);
    const int limit = there ? min(seen, len - n + i + 1) : 0;
    // the tile's last column sees the most
    const int last = min(n_cols - 1, tile * COLS + COLS - 1) / a.group;
    const int end = min(seen, len - n + last + 1);
    const int k0 = chunk * a.chunk, k1 = min(end, k0 + a.chunk);
    if (k0 >= end && chunk) return;

    const int64_t row = fm_seq_row0(b, s) + i;
    Columns<D, NP> w;
    w.template load_q<BF16>(a.q, row * a.q_stride + (int64_t)qh * D, there, a.scale_log2);
    for (int pos = k0 + wave * BK; pos < k1; pos += 4 * BK) w.step(c, s, h, pos, limit);
    w.l += __shfl_xor(w.l, 16);
    w.l += __shfl_xor(w.l, 32);

    // join the waves: wave 0 takes the others' sums at the common maximum
    if (g == 0) s_m[wave][col] = w.m, s_l[wave][col] = w.l;
    __syncthreads();
    const float m = fmaxf(fmaxf(s_m[0][col], s_m[1][col]), fmaxf(s_m[2][col], s_m[3][col]));
    const float base = m == -INFINITY ? 0.0f : m;
    const float f = ldexpf(exp2f(w.m - base), w.ref);
#pragma unroll
    for (int d = 0; d < DT; d++) w.o[d] *= f;
    if (wave) {
#pragma unroll
        for (int d = 0; d < DT; d++) *(fm_v4f *)s_o[wave - 1][d][lane] = w.o[d];
    }
    __syncthreads();
    if (wave || !there) return;
    float l = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; v++) l = fmaf(s_l[v][col], exp2f(s_m[v][col] - base), l);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int v = 0; v < 3; v++) w.o[d] += *(const fm_v4f *)s_o[v][d][lane];
    // register i of tile d: dim 16 d + 4 g + i
    if (a.n_chunks == 1) {
        const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        const int64_t at = (row * a.q_heads + qh) * D + 4 * g;
#pragma unroll
        for (int d = 0; d < DT; d++) fm_st4<BF16>(a.out, at + 16 * d, w.o[d] * inv);
    } else {
        const int64_t at = ((row * a.q_heads + qh) * a.n_chunks + chunk);
#pragma unroll
        for (int d = 0; d < DT; d++) *(fm_v4f *)(a.part_o + at * D + 16 * d + 4 * g) = w.o[d];
        if (g == 0) a.part_ml[2 * at] = m, a.part_ml[2 * at + 1] = l;
    }
}

// joins the chunks of one (row, query head); one wave each, D / 64 dims a lane
template <int D, bool BF16>
__global__ __launch_bounds__(64) void fm_attn_join(FmKv c, FmAttn a, FmSeqs b) {
    const int s = blockIdx.z, i = blockIdx.y, qh = blockIdx.x, lane = threadIdx.x;
    const int n = fm_seq_rows(b, s);
    if (i >= n) return;
    const int len = c.len[s];
    // the chunks that the row's column tile ran
    const int tile = (i * a.group + qh % a.group) / COLS;
    const int last = min(n * a.group - 1, tile * COLS + COLS - 1) / a.group;
    const int end = min(min(len, a.max_len), len - n + last + 1);
    const int chunks = end <= 0 ? 1 : (end + a.chunk - 1) / a.chunk;
    const int64_t row = fm_seq_row0(b, s) + i, at = (row * a.q_heads + qh) * a.n_chunks;
    float m = -INFINITY;
    for (int k = 0; k < chunks; k++) m = fmaxf(m, a.part_ml[2 * (at + k)]);
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[D / 64];
#pragma unroll
    for (int d = 0; d < D / 64; d++) o[d] = 0.0f;
    for (int k = 0; k < chunks; k++) {
        const float f = exp2f(a.part_ml[2 * (at + k)] - base);
        l = fmaf(f, a.part_ml[2 * (at + k) + 1], l);
#pragma unroll
        for (int d = 0; d < D / 64; d++) o[d] = fmaf(f, a.part_o[(at + k) * D + 64 * d + lane], o[d]);
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
#pragma unroll
    for (int d = 0; d < D / 64; d++) fm_st1<BF16>(a.out, (row * a.q_heads + qh) * D + 64 * d + lane, o[d] * inv);
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
// run of tokens is rewritten (its other bytes as they are); fewer than 16 tokens go byte by byte.
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
    const float scale = fmaxf(old, __fdiv_rn(big, 127.0f));
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
void launch_cols(const FmKv &c, const FmAttn &a, const FmSeqs &b, hipStream_t st) {
    hipLaunchKernelGGL((fm_attn_cols<D, BF16>), dim3(a.n_chunks * a.n_tiles, c.kv_heads, b.n_seq), dim3(256), 0, st, c, a, b);
    if (a.n_chunks > 1)
        hipLaunchKernelGGL((fm_attn_join<D, BF16>), dim3(a.q_heads, fm_most_rows(b), b.n_seq), dim3(64), 0, st, c, a, b);
}

}  // namespace

extern "C" int fm_launch_attn(const FmKv *c, FmAttn *a, const FmSeqs *b, int D, int bf16, void *ws, hipStream_t st) {
    if (a->n_tiles < 1) return FM_OK;
    a->part_o = (float *)ws;
    a->part_ml = a->part_o ? a->part_o + (size_t)fm_all_rows(*b) * a->q_heads * a->n_chunks * D : nullptr;
    switch (D) {
        case 64: bf16 ? launch_cols<64, true>(*c, *a, *b, st) : launch_cols<64, false>(*c, *a, *b, st); break;
        case 128: bf16 ? launch_cols<128, true>(*c, *a, *b, st) : launch_cols<128, false>(*c, *a, *b, st); break;
        case 256: bf16 ? launch_cols<256, true>(*c, *a, *b, st) : launch_cols<256, false>(*c, *a, *b, st); break;
        default: return FM_ERR_UNSUPPORTED;
    }
    return hipGetLastError() == hipSuccess ? FM_OK : FM_ERR_HIP;
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
