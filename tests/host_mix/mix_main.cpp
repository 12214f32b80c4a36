// Host program over finchmoe_amd/csrc/fm_mix_index.h: every refusal of the token mixers' entry
// points, and a walk of the paged cache's addresses — each (sequence, head, step, lane, load) of the
// attention and of the appends, over page tables with entries that are not there, against the buffers'
// sizes.  Built with the address and undefined-behaviour sanitizers; no GPU.
#include <stdio.h>
#include <stdlib.h>

#include <set>
#include <vector>

#include "../../finchmoe_amd/csrc/fm_mix_index.h"

static int bad = 0;
#define CHECK(cond)                                                       \
    do {                                                                  \
        if (!(cond)) {                                                    \
            printf("line %d: %s\n", __LINE__, #cond);                     \
            bad++;                                                        \
        }                                                                 \
    } while (0)

static unsigned rnd_state = 1;
static int rnd(int n) {
    rnd_state = rnd_state * 1664525u + 1013904223u;
    return (int)((rnd_state >> 8) % (unsigned)n);
}
static void *at(uintptr_t a) { return (void *)a; }

// ---- refusals
static void refuse_gdn() {
    FmWhy w;
    FmGdn a;
    const uintptr_t B = 1 << 20;
    const float *in[3] = {(float *)at(B), (float *)at(2 * B), nullptr};
    float *out[3] = {(float *)at(B), (float *)at(4 * B), (float *)at(5 * B)};
    int start[4] = {0, 5, 5, 9};
    fm_gated_delta_args g{};
    g.n_seq = 3, g.k_heads = 2, g.v_heads = 4, g.k_dim = 128, g.v_dim = 64, g.scale = 1;
    g.d_q = g.d_k = g.d_v = at(16 * B), g.d_out = at(32 * B), g.d_g = g.d_beta = (float *)at(48 * B);
    g.q_stride = g.k_stride = g.v_stride = 256;
    g.seq_start = start, g.d_state_in = in, g.d_state_out = out;
    CHECK(fm_gdn_check(&w, &g, &a) == FM_OK);
    CHECK(fm_gdn_check(&w, nullptr, &a) == FM_ERR_ARG);
#define BAD(field, value, code)                                           \
    do {                                                                  \
        auto h = g;                                                       \
        h.field = value;                                                  \
        CHECK(fm_gdn_check(&w, &h, &a) == code);                          \
    } while (0)
    BAD(n_seq, 0, FM_ERR_ARG);
    BAD(n_seq, FM_MAX_SEQ + 1, FM_ERR_ARG);
    BAD(k_heads, 0, FM_ERR_ARG);
    BAD(k_heads, 3, FM_ERR_ARG);
    BAD(v_heads, 1, FM_ERR_ARG);
    BAD(v_heads, 512, FM_ERR_ARG);
    BAD(k_dim, 96, FM_ERR_UNSUPPORTED);
    BAD(v_dim, 0, FM_ERR_UNSUPPORTED);
    BAD(v_dim, 40, FM_ERR_UNSUPPORTED);
    BAD(v_dim, 272, FM_ERR_UNSUPPORTED);
    BAD(dtype, 2, FM_ERR_ARG);
    BAD(flags, 2, FM_ERR_ARG);
    BAD(d_q, nullptr, FM_ERR_ARG);
    BAD(d_k, at(16 * B + 8), FM_ERR_ARG);
    BAD(d_out, at(16 * B + 4), FM_ERR_ARG);
    BAD(d_g, nullptr, FM_ERR_ARG);
    BAD(d_beta, (float *)at(B + 2), FM_ERR_ARG);
    BAD(q_stride, 255, FM_ERR_ARG);
    BAD(k_stride, 258, FM_ERR_ARG);
    BAD(v_stride, -256, FM_ERR_ARG);
    BAD(d_state_out, nullptr, FM_ERR_ARG);
    {
        auto h = g;
        h.dtype = FM_DTYPE_BF16;
        h.q_stride = 260;      // 520 bytes: not a multiple of 16
        CHECK(fm_gdn_check(&w, &h, &a) == FM_ERR_ARG);
    }
    int s1[4] = {1, 5, 5, 9}, s2[4] = {0, 5, 4, 9}, s3[4] = {0, 5, 5, 70000};
    BAD(seq_start, s1, FM_ERR_ARG);
    BAD(seq_start, s2, FM_ERR_ARG);
    BAD(seq_start, s3, FM_ERR_ARG);
    const size_t state = 4 * 64 * 128 * 4;
    float *o1[3] = {(float *)at(B), (float *)at(B), (float *)at(5 * B)};
    float *o2[3] = {(float *)at(4 * B), (float *)at(4 * B + state - 16), (float *)at(5 * B)};
    float *o3[3] = {(float *)at(2 * B), (float *)at(4 * B), (float *)at(5 * B)};      // another sequence's input
    float *o4[3] = {(float *)at(B + 16), (float *)at(4 * B), (float *)at(5 * B)};     // its own input, shifted
    float *o5[3] = {(float *)at(B), (float *)at(4 * B), nullptr};
    float *o6[3] = {(float *)at(B + 4), (float *)at(4 * B), (float *)at(5 * B)};
    for (auto o : {o1, o2, o3, o4, o5, o6}) BAD(d_state_out, o, FM_ERR_ARG);
    float *o7[3] = {(float *)at(4 * B + state), (float *)at(4 * B), (float *)at(4 * B + 2 * state)};
    BAD(d_state_out, o7, FM_OK);
    BAD(d_state_in, nullptr, FM_OK);
    BAD(seq_start, nullptr, FM_OK);
#undef BAD
    // the overlap rule against plain pairwise comparison
    for (int round = 0; round < 20000; round++) {
        const int n = 1 + rnd(5);
        const float *ri[5];
        float *ro[5];
        for (int i = 0; i < n; i++) {
            ri[i] = rnd(4) ? (float *)at(B + (uintptr_t)rnd(14) * (state / 2)) : nullptr;
            ro[i] = (float *)at(B + (uintptr_t)rnd(14) * (state / 2));
        }
        bool clash = false;
        auto meet = [&](const void *x, const void *y) { return (uintptr_t)x < (uintptr_t)y + state && (uintptr_t)y < (uintptr_t)x + state; };
        for (int i = 0; i < n; i++)
            for (int j = 0; j < n; j++) {
                if (j < i && meet(ro[i], ro[j])) clash = true;
                if (ri[j] && meet(ro[i], ri[j]) && !(i == j && ro[i] == ri[j])) clash = true;
            }
        auto h = g;
        h.n_seq = n, h.seq_start = nullptr, h.d_state_in = ri, h.d_state_out = ro;
        CHECK((fm_gdn_check(&w, &h, &a) == FM_OK) == !clash);
    }
}

static void refuse_cache() {
    FmWhy w;
    FmKv k;
    FmAttn a;
    FmSeqs b;
    FmKvRows x;
    size_t ws;
    const uintptr_t B = 1 << 20;
    fm_attn_args g{};
    g.cache.d_k = g.cache.d_v = at(B), g.cache.d_k_scale = g.cache.d_v_scale = (float *)at(2 * B);
    g.cache.n_pages = 4, g.cache.page_tokens = 32, g.cache.kv_heads = 2, g.cache.head_dim = 128;
    g.n_seq = 2, g.q_heads = 6, g.scale = 1, g.d_q = at(3 * B), g.d_out = at(4 * B), g.q_stride = 768;
    g.d_len = g.d_pages = (int32_t *)at(5 * B), g.max_pages = 3, g.max_len = 96;
    CHECK(fm_attn_check(&w, &g, 256, &k, &a, &b, &ws) == FM_OK);
    CHECK(fm_attn_check(&w, nullptr, 256, &k, &a, &b, &ws) == FM_ERR_ARG);
#define BAD(field, value, code)                                           \
    do {                                                                  \
        auto h = g;                                                       \
        h.field = value;                                                  \
        CHECK(fm_attn_check(&w, &h, 256, &k, &a, &b, &ws) == code);       \
    } while (0)
    BAD(cache.d_k, nullptr, FM_ERR_ARG);
    BAD(cache.d_v, at(B + 8), FM_ERR_ARG);
    BAD(cache.d_k_scale, (float *)at(B + 2), FM_ERR_ARG);
    BAD(cache.n_pages, 0, FM_ERR_ARG);
    BAD(cache.page_tokens, 8, FM_ERR_UNSUPPORTED);
    BAD(cache.page_tokens, 256, FM_ERR_UNSUPPORTED);
    BAD(cache.head_dim, 192, FM_ERR_UNSUPPORTED);
    BAD(cache.kv_heads, 0, FM_ERR_ARG);
    BAD(cache.kv_heads, 4, FM_ERR_ARG);
    BAD(q_heads, 0, FM_ERR_ARG);
    BAD(q_heads, 2048, FM_ERR_ARG);
    BAD(d_len, nullptr, FM_ERR_ARG);
    BAD(d_pages, nullptr, FM_ERR_ARG);
    BAD(max_pages, 0, FM_ERR_ARG);
    BAD(max_pages, 1 << 26, FM_ERR_ARG);
    BAD(max_len, -1, FM_ERR_ARG);
    BAD(q_stride, 760, FM_ERR_ARG);
    BAD(d_out, at(4 * B + 2), FM_ERR_ARG);
    BAD(dtype, -1, FM_ERR_ARG);
    BAD(n_seq, 257, FM_ERR_ARG);
#undef BAD
    fm_kv_args r{};
    r.cache = g.cache, r.n_seq = 2, r.d_k = r.d_v = at(6 * B), r.k_stride = r.v_stride = 256;
    r.d_len = r.d_pages = g.d_len, r.max_pages = 3;
    CHECK(fm_kv_rows_check(&w, &r, 0, &k, &x, &b) == FM_OK && fm_kv_rows_check(&w, &r, 1, &k, &x, &b) == FM_OK);
    r.dtype = FM_DTYPE_BF16;
    CHECK(fm_kv_rows_check(&w, &r, 0, &k, &x, &b) == FM_OK && fm_kv_rows_check(&w, &r, 1, &k, &x, &b) == FM_ERR_UNSUPPORTED);
    r.v_stride = 128;
    CHECK(fm_kv_rows_check(&w, &r, 0, &k, &x, &b) == FM_ERR_ARG);
    r.v_stride = 256, r.d_v = nullptr;
    CHECK(fm_kv_rows_check(&w, &r, 0, &k, &x, &b) == FM_ERR_ARG);
}

static void refuse_logprobs() {
    FmWhy w;
    void *p = at(1 << 20);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, p, 5, p, p, p, p) == FM_OK);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, nullptr, 0, nullptr, nullptr, nullptr, nullptr) == FM_OK);
    CHECK(fm_logprob_args_check(&w, nullptr, 3, 100, 100, p, 5, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 0, 100, 100, p, 5, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 65536, 100, 100, p, 5, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 99, p, 5, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, p, 33, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 4, 100, p, 5, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, nullptr, 5, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, p, 5, p, p, nullptr, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, p, 0, p, p, p, p) == FM_ERR_ARG);
    CHECK(fm_logprob_args_check(&w, p, 3, 100, 100, p, 5, at((1 << 20) + 2), p, p, p) == FM_ERR_ARG);
}

// ---- attention's steps: shared out once each, the parts of a tile found again by the join
static void share_out(const FmKv &c, const FmAttn &a, const FmSeqs &b, int D, size_t ws) {
    std::vector<int> first(b.n_seq + 1, 0);
    for (int s = 0; s < b.n_seq; s++)
        first[s + 1] = first[s] + c.kv_heads * fm_attn_head_steps(fm_seq_rows(b, s), a.group, a.wide, a.narrow_most, c.len[s], a.max_len);
    const int total = first[b.n_seq], share = fm_attn_share(total, a.groups);
    CHECK((int64_t)share * a.groups >= total);
    CHECK(ws == (size_t)2 * a.groups * fm_attn_cols(a.wide) * (D + 2) * 4 + (FM_MAX_SEQ + 1) * 4);
    std::set<int> written;      // slots of parts
    int seen = 0;
    for (int s = 0; s < b.n_seq; s++) {
        const int n = fm_seq_rows(b, s);
        for (int h = 0; h < c.kv_heads; h++)
            for (int t = 0; t < fm_attn_tiles(n, a.group, a.wide, a.narrow_most); t++) {
                const int steps = fm_attn_steps(n, a.group, a.wide, c.len[s], a.max_len, t), at = seen;
                const int end = fm_attn_end(n, a.group, a.wide, c.len[s], a.max_len, t);
                CHECK(steps >= 1 && end <= steps * FM_ATTN_KEYS && end <= a.max_len && (steps == 1 || end > (steps - 1) * FM_ATTN_KEYS));
                seen += steps;
                const int g0 = at / share, g1 = (at + steps - 1) / share;
                CHECK(g1 < a.groups);
                if (g0 == g1) continue;
                for (int g = g0; g <= g1; g++) {
                    // what the workgroup has of the tile, and where both kernels put it
                    const int lo = g * share > at ? g * share - at : 0;
                    const int slot = fm_attn_slot(g, lo);
                    CHECK(slot == fm_attn_slot(g, g * share - at) && slot < 2 * a.groups);
                    CHECK(written.insert(slot).second);
                }
            }
    }
    CHECK(seen == total);
}

// ---- the cache's addresses
static void walk(int n_seq, int kv, int D, int P, int group) {
    const int n_pages = 1 + rnd(12), max_pages = 1 + rnd(6);
    std::vector<int32_t> table((size_t)n_seq * max_pages), len(n_seq);
    for (auto &t : table) t = rnd(5) ? rnd(n_pages) : rnd(2) ? -1 - rnd(5) : n_pages + rnd(3);
    std::vector<int> start(n_seq + 1, 0);
    for (int s = 0; s < n_seq; s++) {
        len[s] = rnd(8) ? rnd(max_pages * P + 40) : (rnd(2) ? -3 : 0);
        start[s + 1] = start[s] + rnd(rnd(3) ? 70 : 400);
    }
    FmKv c{};
    c.n_pages = n_pages, c.page_tokens = P, c.page_shift = __builtin_ctz((unsigned)P), c.kv_heads = kv;
    c.len = len.data(), c.pages = table.data(), c.max_pages = max_pages;
    const int64_t bytes = (int64_t)n_pages * kv * P * D;
    FmAttn a{};
    a.q_heads = kv * group, a.group = group, a.max_len = rnd(2) ? max_pages * P + 100 : 1 + rnd(max_pages * P);
    FmSeqs b{};
    b.n_seq = n_seq;
    for (int s = 0; s <= n_seq; s++) b.start[s] = start[s];
    int covered = 0;
    const int wide_cols = rnd(2) ? 64 : 128, n_cu = 1 + rnd(64);
    if (rnd(2)) a.wide_cols = wide_cols;      // (short sequences may go with the wide ones)
    for (int wide : {0, wide_cols}) {
        const size_t ws = fm_attn_plan(&c, &a, &b, D, n_cu, wide);
        CHECK(a.max_len <= max_pages * P);
        if (!a.n_tiles) {
            CHECK(ws == 0);
            continue;
        }
        CHECK(a.groups >= 1);
        if (!wide) share_out(c, a, b, D, ws);
        else {
            FmWide w;
            fm_attn_wide_tiles(b, group, wide, a.narrow_most, &w);
            const int tiles = w.first[n_seq] * kv, units = tiles * a.splits;
            CHECK(a.groups <= units && ws == (a.splits == 1 ? 0 : (size_t)units * wide * (D + 2) * 4));
            std::set<int> picked;
            for (int round = 0; round * a.groups < units; round++)
                for (int g = 0; g < a.groups; g++) {
                    const int u = fm_attn_wide_pick(round, g, a.groups);
                    if (u < units) CHECK(picked.insert(u).second);
                }
            CHECK((int)picked.size() == units);
            std::set<std::vector<int>> seen;
            for (int u = 0; u < units; u++) {
                const FmWideUnit at = fm_attn_wide_unit(w, n_seq, kv, a.splits, u);
                CHECK(at.s < n_seq && at.h < kv && at.part < a.splits && at.tile >= 0 && at.tile < fm_attn_tiles(fm_seq_rows(b, at.s), group, wide, a.narrow_most));
                CHECK(seen.insert({at.s, at.h, at.tile, at.part}).second);
                const FmWideUnit one = fm_attn_wide_unit(w, n_seq, kv, a.splits, u / a.splits * a.splits);
                CHECK(one.s == at.s && one.h == at.h && one.tile == at.tile && one.part == 0);
            }
        }
    }
    for (int s = 0; s < n_seq; s++) {      // a sequence's columns are in one of the two launches
        const int n = fm_seq_rows(b, s), narrow = fm_attn_tiles(n, group, 0, a.narrow_most), wides = fm_attn_tiles(n, group, 64, a.narrow_most);
        CHECK(!narrow || !wides);
        CHECK(narrow * FM_ATTN_COLS + wides * 64 >= n * group);
        covered += narrow + wides;
    }
    CHECK(covered >= 0);
    for (int s = 0; s < n_seq; s++)
        for (int h = 0; h < kv; h++)
            // (every step of the table and some behind it)
            for (int pos0 = 0; pos0 < (max_pages * P + 300) / 64 * 64; pos0 += FM_ATTN_KEYS)
                for (int lane = 0; lane < 64; lane++) {
                    const int g = lane >> 4, r = lane & 15;
                    const int kp = fm_kv_page(c, s, pos0 + 16 * (r >> 2)), vp = fm_kv_page(c, s, pos0 + 16 * g);
                    CHECK(kp < n_pages && vp < n_pages);
                    const int64_t kb = fm_kv_k_at(c, D, kp < 0 ? 0 : kp, h, pos0 + 16 * (r >> 2) + (r & 3), 16 * g);
                    const int64_t vb = fm_kv_v_at(c, D, vp < 0 ? 0 : vp, h, pos0 + 16 * g, r);
                    for (int d = 0; d < D / 64; d++)
                        for (int t = 0; t < 4; t++) CHECK(kb + 4 * t * D + 64 * d >= 0 && kb + 4 * t * D + 64 * d + 16 <= bytes);
                    for (int d = 0; d < D / 16; d++) CHECK(vb + (int64_t)16 * d * P >= 0 && vb + (int64_t)16 * d * P + 16 <= bytes);
                    CHECK(kb % 16 == 0 && vb % 16 == 0);
                }
    // appends: every row of a sequence that has a place is written once, to its own place
    const int most = fm_most_rows(b);
    for (int s = 0; s < n_seq; s++) {
        const int n = start[s + 1] - start[s];
        std::set<int> seen;
        for (int j = 0; j < (most + P - 2) / P + 1; j++) {
            FmKvSpan sp;
            if (!fm_kv_span(n, len[s], c.page_shift, j, &sp)) continue;
            CHECK(sp.t0 >= 0 && sp.t0 < sp.t1 && sp.t1 <= P);
            const int page = fm_kv_page(c, s, sp.start);
            for (int t = sp.t0; t < sp.t1; t++) {
                CHECK(sp.row0 + t >= 0 && sp.row0 + t < n && sp.start + t == len[s] - n + sp.row0 + t);
                CHECK(seen.insert(sp.start + t).second);
                if (page < 0) continue;
                for (int d = 0; d < D; d += D - 1) {
                    const int64_t ka = fm_kv_k_at(c, D, page, kv - 1, t, d), va = fm_kv_v_at(c, D, page, kv - 1, t, d);
                    CHECK(ka >= 0 && ka < bytes && va >= 0 && va < bytes);
                }
            }
        }
        CHECK((int)seen.size() == (len[s] <= 0 ? 0 : n < len[s] ? n : len[s]));
    }
}

// ---- the gated delta rule's launches: every row runs once, in order, and the workspace holds a launch
static void plan_gdn() {
    for (int round = 0; round < 3000; round++) {
        FmGdn a{};
        a.k_heads = 1 + rnd(16), a.v_heads = a.k_heads * (1 + rnd(3)), a.k_dim = rnd(2) ? 64 : 128, a.v_dim = 128;
        const int n = 1 + rnd(rnd(4) ? 6 : FM_MAX_SEQ);
        std::vector<int> start(n + 1, 0);
        for (int i = 0; i < n; i++) start[i + 1] = start[i] + (rnd(3) ? rnd(60) : rnd(65536 / n));
        std::vector<float *> in(n), out(n);
        std::vector<int> next(n, 0);
        for (int i = 0; i < n; i++) in[i] = (float *)at(4096 + 64 * i), out[i] = (float *)at(1 << 20 | 64 * i);
        FmGdnPlan plan{&a, start.data(), n, in.data(), out.data()};
        FmGdnSeqs b;
        int chunked;
        const size_t ws = fm_gdn_ws_bytes(&a, start.data(), n);
        while (plan.next(&b, &chunked)) {
            CHECK(b.n >= 1 && b.n <= FM_GDN_SEQS);
            for (int k = 0; k < b.n; k++) {
                const int i = (int)(((uintptr_t)b.out[k] & ((1 << 20) - 1)) / 64);
                CHECK(b.row[k] == start[i] + next[i] && b.in[k] == (next[i] ? out[i] : in[i]));
                CHECK(b.row[k] + b.rows[k] <= start[i + 1]);
                CHECK(chunked == (start[i + 1] - start[i] >= FM_GDN_MIN_CHUNKED));
                CHECK(!chunked || b.rows[k] % FM_GDN_CHUNK == 0 || b.row[k] + b.rows[k] == start[i + 1]);
                next[i] += b.rows[k] ? b.rows[k] : -1;      // (an empty sequence runs once, its state is copied)
                for (int c = b.chunk0[k]; c < b.chunk0[k + 1]; c++) CHECK(fm_gdn_seq_of(b, c) == k);
            }
            if (chunked) CHECK((size_t)b.chunk0[b.n] * fm_gdn_ws(a).floats * 4 <= ws);
        }
        for (int i = 0; i < n; i++) CHECK(next[i] == (start[i + 1] > start[i] ? start[i + 1] - start[i] : -1));
    }
    FmGdn a{};
    a.k_heads = 16, a.v_heads = 32, a.k_dim = a.v_dim = 128;
    CHECK(fm_gdn_ws_bytes(&a, nullptr, 200) == 0);
    const FmGdnWs w = fm_gdn_ws(a);
    CHECK(w.tm % 4 == 0 && w.p % 4 == 0 && w.sc % 4 == 0 && w.floats % 4 == 0 && w.end + a.v_heads <= w.floats);
    CHECK(sizeof(FmGdnSeqs) + sizeof(FmGdn) + 8 <= 4096 && sizeof(FmSeqs) + sizeof(FmKv) + sizeof(FmAttn) + sizeof(FmWide) <= 4096);
}

int main() {
    plan_gdn();
    refuse_gdn();
    refuse_cache();
    refuse_logprobs();
    for (int round = 0; round < 60; round++)
        for (int P : {16, 32, 64, 128}) walk(1 + rnd(4), 1 + rnd(3), 64 << rnd(3), P, 1 + rnd(9));
    // far offsets: past 32 bits
    FmKv c{};
    c.n_pages = 1 << 20, c.page_tokens = 128, c.page_shift = 7, c.kv_heads = 8;
    CHECK(fm_kv_k_at(c, 256, (1 << 20) - 1, 7, 127, 255) == ((int64_t)(1 << 20) * 8 * 128 * 256) - 1);
    CHECK(fm_kv_v_at(c, 256, (1 << 20) - 1, 7, 127, 255) == ((int64_t)(1 << 20) * 8 * 128 * 256) - 1);
    FmKvSpan sp;
    CHECK(fm_kv_span(3, 2147483647, 4, 0, &sp) && !fm_kv_span(3, 2147483647, 4, 1 << 28, &sp));
    if (!bad) printf("all refusals and addresses hold\n");
    return bad ? 1 : 0;
}
