// fm_gdn.hip — the gated delta rule (include/finch_hip.h, fm_gated_delta_dev).
//
// Per value head, with the state S [v_dim][k_dim]:
//   S <- exp(g) S;  u = beta (v - S k);  S <- S + u k^T;  o = scale S q
//
// fm_gdn_steps: token by token.  Sixteen lanes (one DPP row) hold a row of the state, k_dim / 16
// values each, so a wave covers four rows per register set and nothing but the row sums crosses
// lanes.  Both products with the state are taken on the OLD state,
//   S_old k, S_old q, k.q  ->  u = beta (v - e^g S_old k),  o = scale (e^g S_old q + u k.q),
// so the sums of a token (these three and, normalised, |k|^2 and |q|^2) do not wait for each
// other.  The state is read and written once per call and lives in registers in between: a call
// of one token per sequence is bound by that traffic (48 sequences with 32 heads of 128 x 128: 203 MB in 35.4 us,
// 5.7 TB/s; one sequence: 4.2 us, a launch), a longer one by the chain of its sums (0.5 us a token).
//
// Longer sequences run in chunks of C = 64 tokens.  With G_i the sum of the chunk's g up to token i,
// E_ij = e^(G_i - G_j) for j <= i and a chunk's rows K, Q, V, the u of all its tokens solve a triangular system,
//   u_i + beta_i sum_{j<i} E_ij (k_i.k_j) u_j = beta_i (v_i - e^G_i S k_i)    =:  (1 + A) u = R
//   o_i = scale (e^G_i S q_i + sum_{j<=i} E_ij (q_i.k_j) u_j)
//   S <- e^G_C S + sum_i e^(G_C - G_i) u_i k_i^T
// Everything that does not need the state — the inverse T of 1 + A, P = scale tril(E . Q K^T) and the
// factors of a token — is computed for all chunks at once by fm_gdn_prep; fm_gdn_scan walks the chunks in
// order, sixteen state rows (value dims) a workgroup, with five small products a chunk.  Both use
// the fp32 matrix instruction v_mfma_f32_16x16x4_f32, eight of them (256 cycles) for 16 x 16 x 32, and operands as they
// are.  (Three bf16 pieces hold an fp32 number: six products of 16 cycles for fp32 K and Q, three for bf16 ones, which need
// no pieces.  That form has not been built.)
// G is summed in fp64: E_ij is a difference of sums that may be hundreds while it is small itself.
#include "fm_mix.h"

namespace {

template <int DK>
struct RowPart {   // a lane's part of a k_dim vector: elements 4 li .. and, of 128, 64 + 4 li ..
    static constexpr int N = DK / 64;
    fm_v4f p[N];
    // (the state is read once and written once: it is not kept in the caches)
    __device__ __forceinline__ void load(const float *row, int li) {
#pragma unroll
        for (int n = 0; n < N; n++) p[n] = __builtin_nontemporal_load((const fm_v4f *)(row + 64 * n + 4 * li));
    }
    __device__ __forceinline__ void store(float *row, int li) const {
#pragma unroll
        for (int n = 0; n < N; n++) __builtin_nontemporal_store(p[n], (fm_v4f *)(row + 64 * n + 4 * li));
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int n = 0; n < N; n++) p[n] = fm_v4f{0.f, 0.f, 0.f, 0.f};
    }
    __device__ __forceinline__ void update(float decay, float u, const RowPart &k) {
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) p[n][i] = fmaf(u, k.p[n][i], decay * p[n][i]);
    }
    template <bool BF16>
    __device__ __forceinline__ void load_any(const void *base, int64_t at, int li) {
#pragma unroll
        for (int n = 0; n < N; n++) p[n] = fm_ld4<BF16>(base, at + 64 * n + 4 * li);
    }
    __device__ __forceinline__ float dot(const RowPart &o) const {
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) s = fmaf(p[n][i], o.p[n][i], s);
        return s;
    }
};

template <int DK, bool BF16>
__global__ __launch_bounds__(256) void fm_gdn_steps(FmGdn a, FmGdnSeqs b) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15;
    const int s = blockIdx.z, h = blockIdx.y, hk = h / (a.v_heads / a.k_heads);
    const int v0 = 16 * blockIdx.x + 4 * wave + (lane >> 4);         // the lane group's row of the state
    const int t0 = b.row[s], T = b.rows[s];
    const int64_t state_at = ((int64_t)h * a.v_dim + v0) * DK;
    RowPart<DK> st;
    if (b.in[s]) st.load(b.in[s] + state_at, li);
    else st.clear();
    RowPart<DK> k, q, nk, nq;
    float v = 0.f, nv = 0.f, g = 0.f, beta = 0.f, ng = 0.f, nbeta = 0.f;
    auto fetch = [&](int t, RowPart<DK> &kk, RowPart<DK> &qq, float &vv, float &gg, float &bb) {
        const int64_t row = t0 + t;
        kk.template load_any<BF16>(a.k, row * a.k_stride + (int64_t)hk * DK, li);
        qq.template load_any<BF16>(a.q, row * a.q_stride + (int64_t)hk * DK, li);
        vv = fm_ld1<BF16>(a.v, row * a.v_stride + (int64_t)h * a.v_dim + v0);
        gg = a.g[row * a.v_heads + h];
        bb = a.beta[row * a.v_heads + h];
    };
    if (T > 0) fetch(0, k, q, v, g, beta);
    for (int t = 0; t < T; t++) {
        if (t + 1 < T) fetch(t + 1, nk, nq, nv, ng, nbeta);
        float kq = fm_group_sum<16>(k.dot(q)), sk = fm_group_sum<16>(st.dot(k)), sq = fm_group_sum<16>(st.dot(q));
        float kn = 1.0f, qn = a.scale;
        if (a.l2norm) {
            kn = 1.0f / sqrtf(fm_group_sum<16>(k.dot(k)) + 1e-6f);
            qn = a.scale / sqrtf(fm_group_sum<16>(q.dot(q)) + 1e-6f);
        }
        const float decay = expf(g), u = beta * (v - decay * (sk * kn));
        const float o = fmaf(u, kq * (kn * qn), decay * (sq * qn));
        st.update(decay, u * kn, k);
        if (li == 0) fm_st1<BF16>(a.out, ((int64_t)(t0 + t) * a.v_heads + h) * a.v_dim + v0, o);
        k = nk, q = nq, v = nv, g = ng, beta = nbeta;
    }
    st.store(b.out[s] + state_at, li);
}

__device__ __forceinline__ fm_v4f mfma4(float x, float y, fm_v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0);
}
// c += sum over the 4 k of a float4 pair: lane group g supplies k = 4 g + e of each
__device__ __forceinline__ fm_v4f mfma16(fm_v4f x, fm_v4f y, fm_v4f c) {
#pragma unroll
    for (int e = 0; e < 4; e++) c = mfma4(x[e], y[e], c);
    return c;
}

__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = __builtin_amdgcn_readlane((int)(b >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float lane_of(float v, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}

// 2^x by the instruction; results below 2^-126 are 0
__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// (Where the chunks and key heads are fewer than the CUs hold, gridDim.z workgroups share a key head's value
// heads, each with the products of its own: 77 tokens 17 us with one, 12 with two.)
// Per (chunk, key head): K K^T and Q K^T of the chunk's rows, then per value head of the key head the
// decay factors, P, and T = (1 + A)^-1.  T in 16 x 16 blocks: the diagonal ones by forward substitution,
// a column per lane; below them, block column by block column,
//   T_ij = -T_ii sum_{j <= m < i} A_im T_mj,
// where a product's result registers are the next one's right operand as they are (lane 16 g + c has
// rows 4 g .. 4 g + 3 of column c in both), so a block column never leaves its wave's registers.
// 64 chunks of 16 / 32 heads of 128 read and write 180 MB in 50 us, 3.6 TB/s; no unit is busy for more than 29 %, the
// waves of the two workgroups a CU has room for (70 KB of LDS each) wait for 36 %: bound by the phases between the
// barriers, as a few chunks are, 12 us.
template <int DK, bool BF16>
__global__ __launch_bounds__(256) void fm_gdn_prep(FmGdn a, FmGdnSeqs b, float *ws) {
    constexpr int LD = DK + 4, LA = 68;      // rows 4 banks apart: 16 lanes' 16-byte reads do not collide
    // K and Q [64][LD], then K K^T, Q K^T, A (T in its place) and P [64][LA]
    constexpr int ROWS = 2 * 64 * LD > 4 * 64 * LA ? 2 * 64 * LD : 4 * 64 * LA;
    __shared__ __attribute__((aligned(16))) float lds[ROWS];
    __shared__ float norm[2][64];
    float *sk = lds, *sq = lds + 64 * LD, *kk = lds, *qk = lds + 64 * LA, *am = lds + 2 * 64 * LA, *pm = lds + 3 * 64 * LA;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, g = lane >> 4, r = lane & 15;
    const int c = blockIdx.x, hk = blockIdx.y, s = fm_gdn_seq_of(b, c);
    const int first = (c - b.chunk0[s]) * 64, n = min(64, b.rows[s] - first);
    const int64_t row0 = b.row[s] + first;
    const FmGdnWs w = fm_gdn_ws(a);
    float *out = ws + (int64_t)c * w.floats;
    const int rep = a.v_heads / a.k_heads, step = gridDim.z;
    const int64_t gate_at = (row0 + min(lane, n - 1)) * a.v_heads + hk * rep;
    const float *gates = a.g + gate_at, *betas = a.beta + gate_at;
    float next_gate = gates[blockIdx.z], next_beta = betas[blockIdx.z];      // a head ahead
    {
        constexpr int PER = DK / 16;         // float4 of K (and of Q) a thread
        fm_v4f x[2][PER];
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int e = tid + 256 * u, i = e / (DK / 4), d = 4 * (e % (DK / 4));
            const int64_t row = row0 + min(i, n - 1);
            x[0][u] = fm_ld4<BF16>(a.k, row * a.k_stride + (int64_t)hk * DK + d);
            x[1][u] = fm_ld4<BF16>(a.q, row * a.q_stride + (int64_t)hk * DK + d);
        }
#pragma unroll
        for (int u = 0; u < PER; u++) {
            const int e = tid + 256 * u, i = e / (DK / 4), d = 4 * (e % (DK / 4));
            const fm_v4f zero = {0.f, 0.f, 0.f, 0.f};
            *(fm_v4f *)(sk + i * LD + d) = i < n ? x[0][u] : zero;
            *(fm_v4f *)(sq + i * LD + d) = i < n ? x[1][u] : zero;
        }
    }
    __syncthreads();
    // 1 / |k| and scale / |q|: two lanes a row and vector
    {
        const float *x = (tid < 128 ? sk : sq) + (tid & 127) / 2 * LD + (tid & 1) * (DK / 2);
        float sum = 0.0f;
        for (int d = 0; d < DK / 2; d += 4) {
            const fm_v4f y = *(const fm_v4f *)(x + d);
#pragma unroll
            for (int e = 0; e < 4; e++) sum = fmaf(y[e], y[e], sum);
        }
        sum = fm_group_sum<2>(sum);
        const float inv = a.l2norm ? 1.0f / sqrtf(sum + 1e-6f) : 1.0f;
        if (!(tid & 1)) norm[tid >> 7][(tid & 127) >> 1] = tid < 128 ? inv : a.scale * inv;
    }
    // the 10 lower tiles of each product, five a wave
    fm_v4f prod[5];
#pragma unroll
    for (int t = 0; t < 5; t++) {
        const int u = (wave * 5 + t) % 10, i = u < 1 ? 0 : u < 3 ? 1 : u < 6 ? 2 : 3, j = u - i * (i + 1) / 2;
        const float *x = (wave < 2 ? sk : sq) + (16 * i + r) * LD + 4 * g, *y = sk + (16 * j + r) * LD + 4 * g;
        fm_v4f z[4];
#pragma unroll
        for (int e = 0; e < 4; e++) z[e] = fm_v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < DK; d += 16) {
            const fm_v4f p = *(const fm_v4f *)(x + d), q = *(const fm_v4f *)(y + d);
#pragma unroll
            for (int e = 0; e < 4; e++) z[e] = mfma4(p[e], q[e], z[e]);
        }
        prod[t] = (z[0] + z[1]) + (z[2] + z[3]);
    }
    // K and Q in the order of the second kernel
    if (blockIdx.z == 0) {
        float *k = out + w.k + (int64_t)hk * DK * 64, *q = out + w.q + (int64_t)hk * DK * 64;
#pragma unroll
        for (int d = 0; d < DK / 16; d++) {
            const int at = (wave * (DK / 16) + d) * FM_GDN_TILE + 4 * lane;
            *(fm_v4f *)(k + at) = *(const fm_v4f *)(sk + (16 * wave + r) * LD + 16 * d + 4 * g);
            *(fm_v4f *)(q + at) = *(const fm_v4f *)(sq + (16 * wave + r) * LD + 16 * d + 4 * g);
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 5; t++) {
        const int u = (wave * 5 + t) % 10, i = u < 1 ? 0 : u < 3 ? 1 : u < 6 ? 2 : 3, j = u - i * (i + 1) / 2;
        float *z = (wave < 2 ? kk : qk) + (16 * i + 4 * g) * LA + 16 * j + r;
#pragma unroll
        for (int e = 0; e < 4; e++) z[e * LA] = prod[t][e];
    }
    const float rk = norm[0][lane], rq = norm[1][lane];
    for (int hh = blockIdx.z; hh < rep; hh += step) {
        const int h = hk * rep + hh;
        float gate = next_gate, beta = next_beta;
        next_gate = gates[min(hh + step, rep - 1)];
        next_beta = betas[min(hh + step, rep - 1)];
        if (lane >= n) gate = beta = 0.0f;
        // e^-104 is 0 in fp32: a stronger decay, -inf included, is the same factor with finite sums
        if (gate < -104.0f) gate = -104.0f;
        double G = (double)gate * 1.4426950408889634;     // (in powers of two from here on)
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double up = __shfl_up(G, o);
            if (lane >= o) G += up;
        }
        if (wave == 0) {
            // factors of a token: of v, of (K S), of u in the state's update, of (Q S)
            float *sc = out + w.sc + (int64_t)h * 256;
            const float eg = exp2_of((float)G);
            sc[lane] = beta;
            sc[64 + lane] = beta * eg * rk;
            sc[128 + lane] = lane < n ? exp2_of((float)(lane_of(G, 63) - G)) * rk : 0.0f;
            sc[192 + lane] = rq * eg;
            if (lane == 63) out[w.end + h] = eg;
        }
        __syncthreads();                       // the products are there; the last head's T and P are out
        // rows 16 wave .. of A and P, a column per lane
        // (computed for every column and dropped above the diagonal: branches would cost more)
#pragma unroll 4
        for (int ii = 0; ii < 16; ii++) {
            const int i = 16 * wave + ii;
            const float x = kk[i * LA + lane], y = qk[i * LA + lane], e = exp2_of((float)(lane_of(G, i) - G));
            const float ai = lane_of(beta, i) * e * (x * (lane_of(rk, i) * rk)), pi = e * (y * (lane_of(rq, i) * rk));
            am[i * LA + lane] = lane < i ? ai : 0.0f;
            pm[i * LA + lane] = lane <= i ? pi : 0.0f;
        }
        __syncthreads();
        if (wave == 3) {
            // diagonal blocks: lane 16 g + r solves column r of block g
            float *d = am + 16 * g * LA + 16 * g;
            float t[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float x = r == i ? 1.0f : 0.0f, y = 0.0f;
#pragma unroll
                for (int m = 0; m < i; m += 4) {
                    const fm_v4f ai = *(const fm_v4f *)(d + i * LA + m);
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (m + e < i) (e & 1 ? y : x) = fmaf(-ai[e], t[m + e], e & 1 ? y : x);
                }
                t[i] = x + y;
            }
            __builtin_amdgcn_wave_barrier();   // (one wave: its LDS accesses run in order)
#pragma unroll
            for (int i = 0; i < 16; i++) d[i * LA + r] = t[i];
        }
        __syncthreads();
        if (wave < 3) {
            // block column `wave`
            fm_v4f t[4];
            const float *d = am + (16 * wave + 4 * g) * LA + 16 * wave + r;
#pragma unroll
            for (int i = 0; i < 4; i++) t[i] = fm_v4f{0.f, 0.f, 0.f, 0.f};
            const fm_v4f diag = {d[0], d[LA], d[2 * LA], d[3 * LA]};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (i == wave) t[i] = diag;
                if (i <= wave) continue;
                fm_v4f x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int m = 0; m < i; m++)
                    if (m >= wave) x = mfma16(*(const fm_v4f *)(am + (16 * i + r) * LA + 16 * m + 4 * g), t[m], x);
                t[i] = -mfma16(*(const fm_v4f *)(am + (16 * i + r) * LA + 16 * i + 4 * g), x, fm_v4f{0.f, 0.f, 0.f, 0.f});
            }
            lds_barrier();                     // every wave has read A
#pragma unroll
            for (int i = 1; i < 4; i++)
                if (i > wave) {
                    float *z = am + (16 * i + 4 * g) * LA + 16 * wave + r;
#pragma unroll
                    for (int e = 0; e < 4; e++) z[e * LA] = t[i][e];
                }
        } else {
            lds_barrier();
        }
        __syncthreads();
        float *tm = out + w.tm + (int64_t)h * 10 * FM_GDN_TILE, *po = out + w.p + (int64_t)h * 10 * FM_GDN_TILE;
#pragma unroll
        for (int u = 0; u < 5; u++) {
            const int t = wave + 4 * u, v = t % 10, i = v < 1 ? 0 : v < 3 ? 1 : v < 6 ? 2 : 3, j = v - i * (i + 1) / 2;
            *(fm_v4f *)((t < 10 ? tm : po) + v * FM_GDN_TILE + 4 * lane) =
                *(const fm_v4f *)((t < 10 ? am : pm) + (16 * i + r) * LA + 16 * j + 4 * g);
        }
    }
}

// The chunks of a sequence in order, 16 value dims of one head per workgroup: eight waves, two per
// token tile of 16.  Of the state [k_dim][16] a wave keeps a tile of 16 k in registers (k_dim 64: the
// second four keep none).  S, R and u pass through LDS as [column][k or token], so that both the writers
// (four consecutive rows of a result) and the readers (four consecutive k of an operand) move 16
// bytes; K as [token][k], of which K^T u reads columns.  A chunk is three phases
// between barriers,
//   1  waves 0-3: R = beta V - f K S                waves 4-7: half of Q S
//   2  waves 0-3: u = T R                                      the other half
//   3  waves 0-3: S += K^T u, k 0-63                waves 4-7: S += K^T u, k 64-127; P u, the output
// which keep a SIMD's matrix core fed by one wave while the other is at a barrier or moves data.
// Operands are fetched for the next chunk right behind their use, into the registers that become free: the
// loads are spread between the products (issued in one go they hold a wave up for as long as the products
// take) and have a chunk's time to arrive.  Every load is issued on every path (rows behind the last
// one as that one, tiles above the diagonal as the diagonal's, what they give is dropped): one that some path
// skips would make the compiler wait for all.
// Bound by the chain of a chunk's three phases, 3.1 us: 8192 tokens of 32 heads of 128 are 128 chunks, 400 us
// of the call's 474.  The matrix cores are busy for 56 % of the time; without the second waves' work, or T R, or
// the loads a chunk would still take 2.5 to 3.0 us.
template <int DK, bool BF16>
__global__ __launch_bounds__(512, 2) void fm_gdn_scan(FmGdn a, FmGdnSeqs b, const float *ws) {
    constexpr int LS = DK + 4, LU = 68, ND = DK / 16;
    __shared__ __attribute__((aligned(16))) float ss[16 * LS], sr[16 * LU], su[16 * LU], sw[16 * LU], sk[64 * LS], none[4];
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wv & 3, lane = threadIdx.x & 63, g = lane >> 4, r = lane & 15;
    const bool second = wv >= 4;
    const int h = blockIdx.x % a.v_heads, v0 = 16 * (blockIdx.x / a.v_heads), s = blockIdx.y;
    const int hk = h / (a.v_heads / a.k_heads);
    const FmGdnWs w = fm_gdn_ws(a);
    const int T = b.rows[s], chunks = (T + 63) / 64;
    const fm_v4f zero = {0.f, 0.f, 0.f, 0.f};
    // the state's rows [v_dim][k_dim] are the columns here
    const bool keeps = !second || DK == 128;
    const int k_at = wv * 16 + 4 * g;
    const int64_t st_at = ((int64_t)h * a.v_dim + v0 + r) * DK + k_at;
    fm_v4f st = zero;
    if (keeps) {
        if (b.in[s]) st = *(const fm_v4f *)(b.in[s] + st_at);
        *(fm_v4f *)(ss + r * LS + k_at) = st;
    }
    if (threadIdx.x < 4) none[threadIdx.x] = 0.0f;
    const float *in;
    int n_in;
    int64_t row_in;
    auto at_chunk = [&](int c) {
        n_in = min(64, T - 64 * c);
        row_in = b.row[s] + 64 * (int64_t)c;
        in = ws + (int64_t)(b.chunk0[s] + c) * w.floats;
    };
    // uniform base, lane offset
    const unsigned lane4 = 4 * lane;
    const int64_t row_at = (second ? w.q : w.k) + ((int64_t)hk * DK * 64 + wave * ND * FM_GDN_TILE);
    const int64_t low_at = (second ? w.p : w.tm) + (int64_t)h * 10 * FM_GDN_TILE + fm_gdn_lower(wave, 0);
    const unsigned sc_lane = 16 * wave + 4 * g;
    auto ld = [&](int64_t at) { return *(const fm_v4f *)(in + at + lane4); };
    fm_v4f rows[ND], low[4], beta = zero, f0 = zero, f1 = zero;      // K or Q, T or P, factors
    float v[4] = {0.f, 0.f, 0.f, 0.f}, decay;
    auto load_low = [&](int j) { low[j] = ld(low_at + min(j, wave) * FM_GDN_TILE); };
    auto load_rows = [&](int d) { rows[d] = ld(row_at + d * FM_GDN_TILE); };
    auto load_v = [&]() {
        const float *sc = in + w.sc + h * 256;
        beta = *(const fm_v4f *)(sc + sc_lane);
        f0 = *(const fm_v4f *)(sc + 64 + sc_lane);
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = fm_ld1<BF16>(a.v, (row_in + min((int)sc_lane + i, n_in - 1)) * a.v_stride + (int64_t)h * a.v_dim + v0 + r);
    };
    auto load_f1 = [&]() { f1 = *(const fm_v4f *)(in + w.sc + h * 256 + (second ? 192 : 128) + sc_lane); };
    auto load_decay = [&]() { decay = in[w.end + h]; };
    // sum over the tiles j <= wave of the lower tiles; the operand of the others is zero
    auto lower = [&](const float *x, fm_v4f first) {
        fm_v4f u[4] = {first, zero, zero, zero};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const fm_v4f y = *(const fm_v4f *)(j <= wave ? x + r * LU + 16 * j + 4 * g : none);
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = mfma4(low[j][e], y[e], u[e]);
            load_low(j);
        }
        return (u[0] + u[1]) + (u[2] + u[3]);
    };
    auto times_s = [&](int d0, int d1, fm_v4f *x) {
#pragma unroll
        for (int d = 0; d < ND; d++)
            if (d >= d0 && d < d1) {
                const fm_v4f y = *(const fm_v4f *)(ss + r * LS + 16 * d + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = mfma4(rows[d][e], y[e], x[e]);
                load_rows(d);
            }
    };
    auto update = [&]() {
        fm_v4f z[4] = {st * decay, zero, zero, zero};
        load_decay();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const fm_v4f y = *(const fm_v4f *)(sw + r * LU + 16 * j + 4 * g);
            const float *x = sk + (16 * j + 4 * g) * LS + 16 * wv + r;
#pragma unroll
            for (int e = 0; e < 4; e++) z[e] = mfma4(x[e * LS], y[e], z[e]);
        }
        st = (z[0] + z[1]) + (z[2] + z[3]);
        *(fm_v4f *)(ss + r * LS + k_at) = st;
    };
    at_chunk(0);
#pragma unroll
    for (int d = 0; d < ND; d++) load_rows(d);
    load_f1();
    load_decay();
#pragma unroll
    for (int j = 0; j < 4; j++) load_low(j);
    if (!second) load_v();
    // (the first chunk's operands arrive before the loop: its waits then go by the loop's own order of loads)
    __builtin_amdgcn_s_waitcnt(0x0F70);                    // vmcnt(0)
    if (!second) {
        for (int c = 0; c < chunks; c++) {
            const int n = n_in;
            at_chunk(min(c + 1, chunks - 1));
            fm_v4f x[4] = {zero, zero, zero, zero};
            lds_barrier();                                 // S is there, the last chunk's K has been read
#pragma unroll
            for (int d = 0; d < ND; d++) *(fm_v4f *)(sk + (16 * wave + r) * LS + 16 * d + 4 * g) = rows[d];
            times_s(0, ND, x);
            const fm_v4f ks = (x[0] + x[1]) + (x[2] + x[3]);
            fm_v4f rr;
#pragma unroll
            for (int i = 0; i < 4; i++) rr[i] = (int)sc_lane + i < n ? beta[i] * v[i] - f0[i] * ks[i] : 0.0f;
            *(fm_v4f *)(sr + r * LU + sc_lane) = rr;
            load_v();
            lds_barrier();                                 // R is there
            const fm_v4f u = lower(sr, zero);
            *(fm_v4f *)(su + r * LU + sc_lane) = u;
            *(fm_v4f *)(sw + r * LU + sc_lane) = u * f1;
            load_f1();
            lds_barrier();                                 // u is there, S has been read
            update();
        }
    } else {
        for (int c = 0; c < chunks; c++) {
            const int n = n_in;
            const int64_t row0 = row_in + sc_lane;
            at_chunk(min(c + 1, chunks - 1));
            fm_v4f x[4] = {zero, zero, zero, zero};
            lds_barrier();
            times_s(0, ND / 2, x);
            lds_barrier();
            times_s(ND / 2, ND, x);
            lds_barrier();
            if (keeps) update();
            const fm_v4f y = lower(su, f1 * ((x[0] + x[1]) + (x[2] + x[3])));
            load_f1();
#pragma unroll
            for (int i = 0; i < 4; i++)
                if ((int)sc_lane + i < n) fm_st1<BF16>(a.out, ((row0 + i) * a.v_heads + h) * a.v_dim + v0 + r, y[i]);
        }
    }
    if (keeps) *(fm_v4f *)(b.out[s] + st_at) = st;
}

template <int DK, bool BF16>
int launch_seqs(const FmGdn &a, const FmGdnSeqs &b, int chunked, float *ws, int n_cu, hipStream_t st) {
    if (!chunked) {
        hipLaunchKernelGGL((fm_gdn_steps<DK, BF16>), dim3(a.v_dim / 16, a.v_heads, b.n), dim3(256), 0, st, a, b);
    } else {
        const int rep = a.v_heads / a.k_heads, share = 2 * n_cu / (b.chunk0[b.n] * a.k_heads);
        const int z = share < 1 ? 1 : share < rep ? share : rep;
        hipLaunchKernelGGL((fm_gdn_prep<DK, BF16>), dim3(b.chunk0[b.n], a.k_heads, z), dim3(256), 0, st, a, b, ws);
        hipLaunchKernelGGL((fm_gdn_scan<DK, BF16>), dim3(a.v_heads * (a.v_dim / 16), b.n), dim3(512), 0, st, a, b, ws);
    }
    return hipGetLastError() == hipSuccess ? FM_OK : FM_ERR_HIP;
}

}  // namespace

// start: n_seq + 1 row numbers (null: one row per sequence); in, out: n_seq state pointers
extern "C" int fm_launch_gdn(const FmGdn *a, int bf16, const int *start, int n_seq, const float *const *in,
                             float *const *out, void *ws, int n_cu, hipStream_t st) {
    FmGdnPlan plan{a, start, n_seq, in, out};
    FmGdnSeqs b;
    int chunked;
    while (plan.next(&b, &chunked)) {
        int rc;
        if (a->k_dim == 128) rc = bf16 ? launch_seqs<128, true>(*a, b, chunked, (float *)ws, n_cu, st) : launch_seqs<128, false>(*a, b, chunked, (float *)ws, n_cu, st);
        else rc = bf16 ? launch_seqs<64, true>(*a, b, chunked, (float *)ws, n_cu, st) : launch_seqs<64, false>(*a, b, chunked, (float *)ws, n_cu, st);
        if (rc) return rc;
    }
    return FM_OK;
}
