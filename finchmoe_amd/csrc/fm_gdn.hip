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
// of one token per sequence is bound by that traffic, a longer one by the chain of its sums.
#include "fm_mix.h"

namespace {

template <int DK>
struct RowPart {   // a lane's part of a k_dim vector: elements 4 li .. and, of 128, 64 + 4 li ..
    static constexpr int N = DK / 64;
    fm_v4f p[N];
    __device__ __forceinline__ void load(const float *row, int li) {
#pragma unroll
        for (int n = 0; n < N; n++) p[n] = *(const fm_v4f *)(row + 64 * n + 4 * li);
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

template <int DK, bool BF16, int R>
__global__ __launch_bounds__(256) void fm_gdn_steps(FmGdn a, FmGdnSeqs b) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15;
    const int s = blockIdx.z, h = blockIdx.y, hk = h / (a.v_heads / a.k_heads);
    const int v0 = (blockIdx.x * 4 + wave) * 4 * R + (lane >> 4);   // rows v0, v0 + 4, ...
    const int t0 = b.start[s], T = b.start[s + 1] - t0;
    const int64_t head = (int64_t)h * a.v_dim * DK;
    const float *in = b.in[s];
    RowPart<DK> st[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
        if (in && v0 + 4 * r < a.v_dim) st[r].load(in + head + (int64_t)(v0 + 4 * r) * DK, li);
        else
#pragma unroll
            for (int n = 0; n < RowPart<DK>::N; n++) st[r].p[n] = fm_v4f{0.f, 0.f, 0.f, 0.f};
    }
    RowPart<DK> k, q, nk, nq;
    float vv[R], nv[R], g = 0.f, beta = 0.f, ng = 0.f, nbeta = 0.f;
    auto fetch = [&](int t, RowPart<DK> &kk, RowPart<DK> &qq, float *v, float &gg, float &bb) {
        const int64_t row = t0 + t;
        kk.template load_any<BF16>(a.k, row * a.k_stride + (int64_t)hk * DK, li);
        qq.template load_any<BF16>(a.q, row * a.q_stride + (int64_t)hk * DK, li);
#pragma unroll
        for (int r = 0; r < R; r++)
            v[r] = v0 + 4 * r < a.v_dim ? fm_ld1<BF16>(a.v, row * a.v_stride + (int64_t)h * a.v_dim + v0 + 4 * r) : 0.0f;
        gg = a.g[row * a.v_heads + h];
        bb = a.beta[row * a.v_heads + h];
    };
    if (T > 0) fetch(0, k, q, vv, g, beta);
    for (int t = 0; t < T; t++) {
        if (t + 1 < T) fetch(t + 1, nk, nq, nv, ng, nbeta);
        float kq = k.dot(q), kk = 1.0f, qq = 1.0f;
        float sk[R], sq[R];
#pragma unroll
        for (int r = 0; r < R; r++) sk[r] = st[r].dot(k), sq[r] = st[r].dot(q);
        kq = fm_group_sum<16>(kq);
        float kn = 1.0f, qn = a.scale;
        if (a.l2norm) {
            kk = fm_group_sum<16>(k.dot(k));
            qq = fm_group_sum<16>(q.dot(q));
            kn = 1.0f / sqrtf(kk + 1e-6f);
            qn = a.scale / sqrtf(qq + 1e-6f);
        }
        const float decay = expf(g);
        kq *= kn * qn;
#pragma unroll
        for (int r = 0; r < R; r++) {
            sk[r] = fm_group_sum<16>(sk[r]) * kn;
            sq[r] = fm_group_sum<16>(sq[r]) * qn;
            const float u = beta * (vv[r] - decay * sk[r]);
            const float o = fmaf(u, kq, decay * sq[r]);
            const float uk = u * kn;
#pragma unroll
            for (int n = 0; n < RowPart<DK>::N; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) st[r].p[n][i] = fmaf(uk, k.p[n][i], decay * st[r].p[n][i]);
            if (li == 0 && v0 + 4 * r < a.v_dim)
                fm_st1<BF16>(a.out, ((int64_t)(t0 + t) * a.v_heads + h) * a.v_dim + v0 + 4 * r, o);
        }
        k = nk, q = nq, g = ng, beta = nbeta;
#pragma unroll
        for (int r = 0; r < R; r++) vv[r] = nv[r];
    }
    float *out = b.out[s];
#pragma unroll
    for (int r = 0; r < R; r++)
        if (v0 + 4 * r < a.v_dim)
#pragma unroll
            for (int n = 0; n < RowPart<DK>::N; n++)
                *(fm_v4f *)(out + head + (int64_t)(v0 + 4 * r) * DK + 64 * n + 4 * li) = st[r].p[n];
}

template <int DK, bool BF16>
void launch_steps(const FmGdn &a, const FmGdnSeqs &b, hipStream_t st) {
    hipLaunchKernelGGL((fm_gdn_steps<DK, BF16, 1>), dim3(a.v_dim / 16, a.v_heads, b.n), dim3(256), 0, st, a, b);
}

}  // namespace

extern "C" size_t fm_gdn_ws_bytes(const FmGdn *, const int *, int) { return 0; }

// start: n_seq + 1 row numbers (null: one row per sequence); in, out: n_seq state pointers
extern "C" int fm_launch_gdn(const FmGdn *a, int bf16, const int *start, int n_seq, const float *const *in,
                             float *const *out, void *ws, int n_cu, hipStream_t st) {
    (void)ws; (void)n_cu;
    for (int first = 0; first < n_seq; first += FM_GDN_SEQS) {
        FmGdnSeqs b;
        b.n = n_seq - first < FM_GDN_SEQS ? n_seq - first : FM_GDN_SEQS;
        for (int i = 0; i <= b.n; i++) b.start[i] = start ? start[first + i] : first + i;
        for (int i = 0; i < b.n; i++) {
            b.in[i] = in ? in[first + i] : nullptr;
            b.out[i] = out[first + i];
        }
        if (a->k_dim == 128) {
            if (bf16) launch_steps<128, true>(*a, b, st);
            else launch_steps<128, false>(*a, b, st);
        } else {
            if (bf16) launch_steps<64, true>(*a, b, st);
            else launch_steps<64, false>(*a, b, st);
        }
        if (hipGetLastError() != hipSuccess) return FM_ERR_HIP;
    }
    return FM_OK;
}
