// Host program over finchmoe_amd/csrc/fm_mix_index.h: how the token mixers' calls are cut into launches.  Each part
// is named on the command line, see tests/test_host_mix_plans.py.  No GPU.
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <string>
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

static unsigned rnd_state = 7;
static int rnd(int n) {
    rnd_state = rnd_state * 1664525u + 1013904223u;
    return (int)((rnd_state >> 8) % (unsigned)n);
}
static void *at(uintptr_t a) { return (void *)a; }

// ---- attention: the steps of a call are counted in 32 bits on the device, whatever its lengths turn out to be
static void count_steps() {
    FmWhy w;
    FmKv k;
    FmAttn a;
    FmSeqs b;
    size_t ws;
    const uintptr_t B = 1 << 20;
    fm_attn_args g{};
    g.cache.d_k = g.cache.d_v = at(B), g.cache.d_k_scale = g.cache.d_v_scale = (float *)at(2 * B);
    g.cache.n_pages = 4, g.cache.page_tokens = 128, g.cache.head_dim = 64;
    g.scale = 1, g.d_q = at(3 * B), g.d_out = at(4 * B), g.d_len = g.d_pages = (int32_t *)at(5 * B);
    int refused = 0, taken = 0;
    for (int round = 0; round < 4000; round++) {
        g.n_seq = 1 + rnd(FM_MAX_SEQ);
        g.cache.kv_heads = 1 << rnd(9);
        g.q_heads = g.cache.kv_heads * (1 + rnd(4));
        if (g.q_heads > 1024) g.q_heads = g.cache.kv_heads;
        g.q_stride = (int64_t)g.q_heads * 64;
        g.max_pages = 1 << rnd(24);
        g.max_len = rnd(4) ? 1 << 30 : 1 + rnd(1 << 20);
        std::vector<int> start(g.n_seq + 1, 0);
        for (int i = 0; i < g.n_seq; i++) start[i + 1] = start[i] + rnd(rnd(3) ? 3 : 200);
        g.seq_start = rnd(2) ? start.data() : nullptr;
        const int rc = fm_attn_check(&w, &g, 256, &k, &a, &b, &ws);
        // all sequences as long as they may be
        int64_t all = 0;
        FmAttn n = a;
        fm_attn_plan(&k, &n, &b, 64, 256, 0);
        for (int s = 0; s < g.n_seq && n.n_tiles; s++) {
            const int rows = fm_seq_rows(b, s);
            for (int t = 0; t < fm_attn_tiles(rows, n.group, 0, n.narrow_most); t++)
                all += (int64_t)k.kv_heads * fm_attn_steps(rows, n.group, 0, n.max_len, n.max_len, t);
        }
        if (rc == FM_OK) {
            taken++;
            CHECK(all <= (1 << 30));
        } else {
            refused++;
            CHECK(rc == FM_ERR_ARG && all + g.n_seq * (int64_t)k.kv_heads * 64 > (1 << 30));
        }
    }
    CHECK(refused > 20 && taken > 2000);
}

// ---- attention: every column of every sequence with rows is in one tile of one of the two launches
static void columns() {
    int both = 0, only_wide = 0, only_narrow = 0;
    for (int round = 0; round < 4000; round++) {
        FmKv c{};
        c.kv_heads = 1 + rnd(8), c.max_pages = 1 + rnd(rnd(2) ? 20 : 600), c.page_tokens = 16 << rnd(4);
        FmAttn a{};
        a.group = 1 + rnd(rnd(2) ? 4 : 16), a.q_heads = a.group * c.kv_heads, a.wide_cols = fm_attn_wide_cols(rnd(2));
        a.max_len = rnd(3) ? c.max_pages * c.page_tokens : rnd(300);
        FmSeqs b{};
        b.n_seq = 1 + rnd(rnd(2) ? 5 : 40), b.one_row = !rnd(5);
        for (int i = 0; i < b.n_seq; i++) b.start[i + 1] = b.start[i] + (rnd(2) ? rnd(3) : rnd(600));
        FmAttn narrow = a, wide = a;
        fm_attn_plan(&c, &narrow, &b, 128, 256, 0);
        fm_attn_plan(&c, &wide, &b, 128, 256, a.wide_cols);
        CHECK(narrow.narrow_most == wide.narrow_most);
        both += narrow.n_tiles && wide.n_tiles, only_wide += !narrow.n_tiles && wide.n_tiles, only_narrow += narrow.n_tiles && !wide.n_tiles;
        FmWide w;
        fm_attn_wide_tiles(b, a.group, a.wide_cols, wide.narrow_most, &w);
        std::vector<std::vector<int>> seen(b.n_seq * c.kv_heads);
        for (int s = 0; s < b.n_seq; s++)
            for (int h = 0; h < c.kv_heads; h++) seen[s * c.kv_heads + h].assign(fm_seq_rows(b, s) * a.group, 0);
        auto mark = [&](int s, int h, int tile, int width) {
            auto &v = seen[s * c.kv_heads + h];
            CHECK(tile * width < (int)v.size());
            for (int k = tile * width; k < (tile + 1) * width && k < (int)v.size(); k++) v[k]++;
        };
        for (int s = 0; s < b.n_seq && narrow.n_tiles; s++)
            for (int h = 0; h < c.kv_heads; h++)
                for (int t = 0; t < fm_attn_tiles(fm_seq_rows(b, s), a.group, 0, narrow.narrow_most); t++) mark(s, h, t, FM_ATTN_COLS);
        for (int u = 0; wide.n_tiles && u < w.first[b.n_seq] * c.kv_heads; u++) {
            const FmWideUnit at = fm_attn_wide_unit(w, b.n_seq, c.kv_heads, 1, u);
            mark(at.s, at.h, at.tile, a.wide_cols);
        }
        for (auto &v : seen)
            for (int n : v) CHECK(n == 1);
    }
    CHECK(both > 100 && only_wide > 100 && only_narrow > 100);
}

// ---- the gated delta rule: long sequences' chunks run in launches that fill a workspace of 192 MB, however the
// lengths differ, and none takes more
struct Launches {
    int n = 0;
    size_t most = 0;      // bytes of the largest
};
static Launches run_gdn(const FmGdn &a, const std::vector<int> &rows) {
    const int n = (int)rows.size();
    std::vector<int> start(n + 1, 0), next(n, 0);
    std::vector<float *> in(n), out(n);
    for (int i = 0; i < n; i++) {
        start[i + 1] = start[i] + rows[i];
        in[i] = (float *)at(4096 + 64 * i), out[i] = (float *)at(1 << 20 | 64 * i);
    }
    FmGdnPlan plan{&a, start.data(), n, in.data(), out.data()};
    FmGdnSeqs b;
    int chunked;
    Launches all;
    while (plan.next(&b, &chunked)) {
        CHECK(b.n >= 1 && b.n <= FM_GDN_SEQS);
        for (int k = 0; k < b.n; k++) {
            const int i = (int)(((uintptr_t)b.out[k] & ((1 << 20) - 1)) / 64);
            CHECK(b.row[k] == start[i] + next[i] && b.in[k] == (next[i] ? out[i] : in[i]) && b.row[k] + b.rows[k] <= start[i + 1]);
            CHECK(!chunked || b.rows[k] % FM_GDN_CHUNK == 0 || b.row[k] + b.rows[k] == start[i + 1]);
            next[i] += b.rows[k];
        }
        if (!chunked) continue;
        all.n++;
        all.most = std::max(all.most, (size_t)b.chunk0[b.n] * fm_gdn_ws(a).floats * 4);
    }
    for (int i = 0; i < n; i++) CHECK(next[i] == rows[i]);
    CHECK(all.most == fm_gdn_ws_bytes(&a, start.data(), n));
    return all;
}
static void windows() {
    FmGdn a{};
    a.k_heads = 16, a.v_heads = 32, a.k_dim = a.v_dim = 128;
    CHECK(run_gdn(a, {8192}).n == 2);
    // a long prompt beside short ones
    for (int others : {1, 7, 31, 100}) {
        std::vector<int> rows(1, 8192);
        rows.insert(rows.end(), others, others == 100 ? 24 : 64);
        CHECK(run_gdn(a, rows).n <= 3);
        std::reverse(rows.begin(), rows.end());
        CHECK(run_gdn(a, rows).n <= 3);
    }
    const size_t full = (size_t)192 << 20;
    a.k_heads = a.v_heads = 256, a.v_dim = 256;
    CHECK(run_gdn(a, std::vector<int>(128, 64)).most <= full);
    for (int round = 0; round < 3000; round++) {
        a.k_heads = 1 + rnd(rnd(2) ? 16 : 256), a.v_heads = std::min(256 / a.k_heads, 1 + rnd(3)) * a.k_heads, a.k_dim = rnd(2) ? 64 : 128, a.v_dim = 128;
        std::vector<int> rows(1 + rnd(rnd(3) ? 8 : FM_MAX_SEQ));
        int left = FM_MAX_ROWS;
        int64_t chunks = 0, many = 0;
        for (int &r : rows) {
            r = std::min(left, rnd(3) ? rnd(200) : rnd(rnd(2) ? 3000 : 20000));
            left -= r;
            if (r >= FM_GDN_MIN_CHUNKED) chunks += (r + FM_GDN_CHUNK - 1) / FM_GDN_CHUNK, many++;
        }
        const int64_t budget = (int64_t)full / (fm_gdn_ws(a).floats * 4);
        const Launches got = run_gdn(a, rows);
        CHECK(got.most <= full);
        // (a launch that ends no sequence fills more than half of the budget, or has FM_GDN_SEQS of them)
        CHECK(got.n <= 1 + 2 * (chunks + budget - 1) / budget + many / FM_GDN_SEQS * 2);
    }
}

int main(int argc, char **argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "steps") count_steps();
    else if (what == "columns") columns();
    else if (what == "windows") windows();
    else bad = 1;
    if (!bad) printf("plans hold\n");
    return bad ? 1 : 0;
}
