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

int main(int argc, char **argv) {
    const std::string what = argc > 1 ? argv[1] : "";
    if (what == "steps") count_steps();
    else bad = 1;
    if (!bad) printf("plans hold\n");
    return bad ? 1 : 0;
}
