// fm_mix_index.h — operands of the token mixers' launches (fm_gdn.hip, fm_attn.hip), the checks
// their entry points make and the index arithmetic of the paged cache, in code that compiles into
// the library, into the kernels and into a plain host program: tests/host_mix/ runs the checks on every
// refusal and walks the cache's addresses without a GPU.
#pragma once

#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <utility>

#include "../../include/finch_hip.h"
#include "fm_index.h"

// rows of one call of a token mixer or of the log probabilities (grid dimensions)
#define FM_MAX_ROWS 65535

// Rows of the sequences of one call.  Passed to kernels by value (kernel arguments hold 4 KB;
// FM_MAX_SEQ + 1 starts are 1 KB), so nothing has to be copied to the device before a launch and a
// captured graph carries its own.  one_row: sequence s is row s.
struct FmSeqs {
    int n_seq, one_row;
    int start[FM_MAX_SEQ + 1];
};
FM_HD int fm_seq_row0(const FmSeqs &s, int i) { return s.one_row ? i : s.start[i]; }
FM_HD int fm_seq_rows(const FmSeqs &s, int i) { return s.one_row ? 1 : s.start[i + 1] - s.start[i]; }

struct FmGdn {
    int k_heads, v_heads, k_dim, v_dim, l2norm;
    float scale;
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const float *g, *beta;
    void *out;
};

// The sequences of one launch, by value: 128 of them are 3.6 KB of kernel arguments.  The launch
// runs rows row[i] .. row[i] + rows[i] - 1; chunk0[i]: chunks of the sequences before (chunked form).
#define FM_GDN_SEQS 128
struct FmGdnSeqs {
    int n;
    int row[FM_GDN_SEQS], rows[FM_GDN_SEQS], chunk0[FM_GDN_SEQS + 1];
    const float *in[FM_GDN_SEQS];
    float *out[FM_GDN_SEQS];
};
// the sequence that chunk `c` of the launch belongs to
FM_HD int fm_gdn_seq_of(const FmGdnSeqs &b, int c) {
    int lo = 0, hi = b.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (b.chunk0[mid] <= c) lo = mid;
        else hi = mid;
    }
    return lo;
}

#define FM_GDN_CHUNK 64
// Sequences of fewer rows run token by token.  Measured (token by token / in chunks, us; 16 key and 32 value heads
// of 128, bf16 alike): one sequence of 24 rows 18.6 / 19.0, of 32 22.7 / 18.9; eight sequences of 24 rows
// 60.5 / 59.7.
#define FM_GDN_MIN_CHUNKED 24
// What the chunked form keeps per chunk between its two kernels, in floats: K and Q of a key head,
// the lower tiles of T and P of a value head, each in the order the second kernel's lanes take them — tiles of 16
// x 16 in 64 groups of four floats, lane 16 g + r has columns 4 g .. 4 g + 3 of row r — then four
// factors per token (sc) and one per chunk (end) of a value head.
struct FmGdnWs {
    int64_t k, q, tm, p, sc, end, floats;
};
#define FM_GDN_TILE 256     // floats
// tile (i, j <= i) of the lower tiles of a 64 x 64 matrix
FM_HDC int fm_gdn_lower(int i, int j) { return (i * (i + 1) / 2 + j) * FM_GDN_TILE; }
FM_HD FmGdnWs fm_gdn_ws(const FmGdn &a) {
    FmGdnWs w;
    const int64_t rows = (int64_t)a.k_heads * a.k_dim * 64, low = (int64_t)a.v_heads * 10 * FM_GDN_TILE;
    w.k = 0;
    w.q = rows;
    w.tm = 2 * rows;
    w.p = w.tm + low;
    w.sc = w.p + low;
    w.end = w.sc + (int64_t)a.v_heads * 256;
    w.floats = w.end + (a.v_heads + 63) / 64 * 64;
    return w;
}
// Chunks of one launch of the chunked form: the workspace stays within 192 MB, where the last-level cache
// still holds it between the two kernels.
inline int fm_gdn_budget(const FmGdn &a) {
    const int64_t n = ((int64_t)192 << 20) / (fm_gdn_ws(a).floats * 4);
    return n < 1 ? 1 : n > (1 << 20) ? 1 << 20 : (int)n;
}
// The launches of a call, in order: next(&seqs, &chunked) fills one, false when there are no more.  The first
// are those of the short sequences.  One of the long ones takes the first of them that have not ended, as many as a launch
// has room for, and of each the chunks left or, if that is too many, the same number: the largest that fits.
struct FmGdnPlan {
    const FmGdn *a;
    const int *start;
    int n_seq;
    const float *const *in;
    float *const *out;
    int at = 0;                     // next sequence to look at
    int pass = 0;                   // 0: short sequences, 1: chunked
    int done[FM_MAX_SEQ] = {};      // chunks of a long sequence that have run
    int rows(int i) const { return start ? start[i + 1] - start[i] : 1; }
    int left(int i) const { return rows(i) < FM_GDN_MIN_CHUNKED ? 0 : (rows(i) + FM_GDN_CHUNK - 1) / FM_GDN_CHUNK - done[i]; }
    bool next(FmGdnSeqs *b, int *chunked) {
        b->n = 0;
        if (pass == 0) {
            for (; at < n_seq && b->n < FM_GDN_SEQS; at++)
                if (rows(at) < FM_GDN_MIN_CHUNKED) put(b, at, 0, rows(at), true);
            *chunked = 0;
            if (b->n) return true;
            pass = 1;
            at = 0;
        }
        *chunked = 1;
        const int budget = fm_gdn_budget(*a);
        while (at < n_seq && !left(at)) at++;
        int seqs[FM_GDN_SEQS], n = 0, most = 0, least = 0, all = 0;
        bool whole = true;                 // these are all that are left
        for (int i = at; i < n_seq; i++) {
            const int c = left(i);
            if (!c) continue;
            if (n == FM_GDN_SEQS || n == budget) {
                whole = false;
                break;
            }
            seqs[n++] = i;
            all += c;
            most = std::max(most, c);
            least = n == 1 ? c : std::min(least, c);
        }
        if (!n) return false;
        int win = 1, over = most + 1;      // win fits, `over` does not or is not needed
        while (over - win > 1) {
            const int mid = (win + over) / 2;
            int64_t sum = 0;
            for (int k = 0; k < n; k++) sum += std::min(left(seqs[k]), mid);
            (sum <= budget ? win : over) = mid;
        }
        // Launches of one size rather than a short last one, where that makes no more of them: to the end of all that
        // are left, or to that of the shortest in hand.
        const int to = whole && (most + win - 1) / win == (all + budget - 1) / budget ? most : least;
        if (to > win) {
            const int passes = (to + win - 1) / win;
            win = (to + passes - 1) / passes;
        }
        for (int k = 0; k < n; k++) {
            const int i = seqs[k], first = done[i] * FM_GDN_CHUNK, c = std::min(left(i), win);
            put(b, i, first, std::min(rows(i) - first, c * FM_GDN_CHUNK), done[i] == 0);
            done[i] += c;
        }
        return true;
    }
    void put(FmGdnSeqs *b, int i, int first, int n, bool fresh) {
        const int k = b->n++;
        b->row[k] = (start ? start[i] : i) + first;
        b->rows[k] = n;
        if (!k) b->chunk0[0] = 0;
        b->chunk0[k + 1] = b->chunk0[k] + (n + FM_GDN_CHUNK - 1) / FM_GDN_CHUNK;
        b->in[k] = fresh ? (in ? in[i] : nullptr) : out[i];
        b->out[k] = out[i];
    }
};
// workspace of a call: that of its largest launch
inline size_t fm_gdn_ws_bytes(const FmGdn *a, const int *start, int n_seq) {
    float *none[FM_MAX_SEQ] = {};
    FmGdnPlan plan{a, start, n_seq, nullptr, none};
    FmGdnSeqs b;
    int chunked, most = 0;
    while (plan.next(&b, &chunked))
        if (chunked && b.chunk0[b.n] > most) most = b.chunk0[b.n];
    return (size_t)most * fm_gdn_ws(*a).floats * sizeof(float);
}

struct FmKv {
    int8_t *k, *v;
    float *k_scale, *v_scale;
    int n_pages, page_tokens, page_shift, kv_heads;
    const int32_t *len, *pages;
    int max_pages;
};

struct FmKvRows {
    const void *k, *v;      // rows appended
    float *k_out, *v_out;   // rows read back
    int64_t k_stride, v_stride;
};

struct FmAttn {
    const void *q;
    int64_t q_stride;
    void *out;
    int q_heads, group;     // query heads per cache head
    float scale_log2;       // scale * log2(e)
    int max_len;            // keys from here on are not seen, at most max_pages * page_tokens
    int wide;               // columns of a wide tile; 0: the launch of the sequences that have narrow ones
    int narrow_most;        // columns of a sequence up to which its tiles are narrow
    int wide_cols;          // columns of the type's wide tiles
    int n_tiles;            // column tiles of the launch's sequence with the most rows
    int groups;             // workgroups that share the steps
    float *part_o, *part_ml;
    int *first;             // narrow tiles: steps before each sequence, for the join
    int splits;             // wide tiles: parts that a tile's steps are cut into
};
#define FM_ATTN_KEYS 64     // keys of a wave's step
#define FM_ATTN_WAVES 4     // waves of a narrow tile's workgroup
#define FM_ATTN_MOST_STEPS (1 << 30)
#define FM_ATTN_COLS 16     // columns of a narrow tile: its waves take different keys
// columns of a wide one, whose queries lie in LDS: fp32 ones as two pieces
FM_HDC int fm_attn_wide_cols(int bf16) { return bf16 ? 128 : 64; }
// Which sequences have wide tiles: those of more than 48 columns, in a batch of 1024 columns over all its
// sequences and cache heads.  Narrow tiles read the keys once per 16 columns but spread over the whole
// chip; measured (narrow / wide, us; 2 cache heads of 256): one sequence over 4000 keys 256 columns
// 33 / 34 (fp32) and 32 / 39 (bf16), 512 columns 44 / 34 and 43 / 40, 1024 columns 68 / 41 and 67 / 42;
// 16 sequences over 3000 keys 32 columns 37 / 32 and 36 / 41, 64 columns 50 / 35 and 49 / 43.
// Beside wide ones the narrow tiles' two launches cost more than wide tiles for all where those are short: one
// sequence of 300 rows and single rows, 2 cache heads of 256 (wide for all / separate, us; by the steps a workgroup then has):
// bf16 3 steps 32 / 46, 8 46 / 50 and 48 / 55, 11 56 / 57, 42 161 / 74; fp32 11 42 / 44, 16 54 / 51, 21 67 / 53.
#define FM_ATTN_NARROW_MOST 48
#define FM_ATTN_WIDE_LEAST 1024
#define FM_ATTN_MIXED_STEPS 12

// ---- attention's steps and who takes them --------------------------------------------------
// A sequence of n rows has n * group columns per cache head (row * group + query head of the group) in
// tiles of 16 or (wide) 64 or 128; a tile's steps are those of 64 keys up to the last one its last column sees, at least
// one (somebody has to write the zeros of a row that sees nothing).
FM_HD int fm_attn_cols(int wide) { return wide ? wide : FM_ATTN_COLS; }
FM_HD int fm_attn_tiles(int n, int group, int wide, int narrow_most) {
    if ((n * group > narrow_most) != (wide != 0)) return 0;
    return (n * group + fm_attn_cols(wide) - 1) / fm_attn_cols(wide);
}
FM_HD int fm_attn_end(int n, int group, int wide, int len, int max_len, int tile) {
    const int cols = n * group, col = (tile + 1) * fm_attn_cols(wide) - 1;
    const int last = (col < cols - 1 ? col : cols - 1) / group, seen = len < max_len ? len : max_len;
    const int end = len - n + last + 1;
    return end < seen ? end : seen;
}
FM_HD int fm_attn_steps(int n, int group, int wide, int len, int max_len, int tile) {
    const int end = fm_attn_end(n, group, wide, len, max_len, tile);
    return end <= FM_ATTN_KEYS ? 1 : (end + FM_ATTN_KEYS - 1) / FM_ATTN_KEYS;
}
// all tiles of one cache head
FM_HD int fm_attn_head_steps(int n, int group, int wide, int narrow_most, int len, int max_len) {
    int sum = 0;
    for (int t = 0; t < fm_attn_tiles(n, group, wide, narrow_most); t++) sum += fm_attn_steps(n, group, wide, len, max_len, t);
    return sum;
}
// Steps are numbered sequence by sequence, head by head, tile by tile; workgroup g takes those from
// g * share on.  A share is at least one step per wave.
FM_HD int fm_attn_share(int total, int groups) {
    const int s = (total + groups - 1) / groups;
    return s < FM_ATTN_WAVES ? FM_ATTN_WAVES : s;
}
// Where a workgroup leaves its part of a tile that it does not have whole: only its first tile can
// have begun in an earlier workgroup, only its last can end in a later one.
FM_HD int fm_attn_slot(int group, int first_step) { return 2 * group + (first_step > 0 ? 0 : 1); }

// ---- the paged cache's addresses -----------------------------------------------------------
// the page that holds position `pos` of sequence s, or -1 for one that is not there
FM_HD int fm_kv_page(const FmKv &c, int s, int pos) {
    if (pos < 0) return -1;
    const int at = pos >> c.page_shift;
    if (at >= c.max_pages) return -1;
    const int p = c.pages[(int64_t)s * c.max_pages + at];
    return p >= 0 && p < c.n_pages ? p : -1;
}
// byte offset of a code: keys [page][head][token][dim], values [page][head][dim][token]
// (A shift for the values' page size: 2048 rows over 8192 keys 403 us in bf16, 410 with a 64-bit product.  One for the
// keys' makes that 406, and 513 of 526 us in fp32; single rows take the same time.)
FM_HD int64_t fm_kv_k_at(const FmKv &c, int D, int page, int head, int pos, int dim) {
    return (((int64_t)page * c.kv_heads + head) * c.page_tokens + (pos & (c.page_tokens - 1))) * D + dim;
}
FM_HD int64_t fm_kv_v_at(const FmKv &c, int D, int page, int head, int pos, int dim) {
    return ((((int64_t)page * c.kv_heads + head) * D + dim) << c.page_shift) + (pos & (c.page_tokens - 1));
}
// Rows of one sequence that an append writes into its j-th page from the first one touched:
// false if there are none.  start: the page's first position; tokens t0 .. t1 - 1 of it; row0: row
// (of the sequence) of the page's token 0, may be negative.
struct FmKvSpan {
    int start, t0, t1, row0;
};
FM_HD bool fm_kv_span(int n, int len, int page_shift, int j, FmKvSpan *out) {
    if (n <= 0 || len <= 0) return false;
    const int first = len < n ? 0 : len - n, P = 1 << page_shift;
    const int64_t start = ((int64_t)(first >> page_shift) + j) << page_shift;
    if (start >= len) return false;
    out->start = (int)start;
    out->t0 = first > out->start ? first - out->start : 0;
    out->t1 = len - out->start < P ? len - out->start : P;
    out->row0 = n - len + out->start;
    return true;
}

// ---- the checks ----------------------------------------------------------------------------
struct FmWhy {
    char text[256];
};
inline int fm_why(FmWhy *w, int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(w->text, sizeof w->text, fmt, ap);
    va_end(ap);
    return code;
}

// Rows of a call's sequences: the check of seq_start that every mixer makes.
inline int fm_check_rows(FmWhy *w, const int32_t *start, int n_seq, int *rows) {
    if (n_seq < 1 || n_seq > FM_MAX_SEQ) return fm_why(w, FM_ERR_ARG, "n_seq %d outside 1..%d", n_seq, FM_MAX_SEQ);
    *rows = n_seq;
    if (!start) return FM_OK;
    if (start[0] != 0) return fm_why(w, FM_ERR_ARG, "seq_start[0] is %d, not 0", start[0]);
    for (int i = 0; i < n_seq; i++)
        if (start[i + 1] < start[i]) return fm_why(w, FM_ERR_ARG, "seq_start[%d] %d below its predecessor %d", i + 1, start[i + 1], start[i]);
    *rows = start[n_seq];
    if (*rows > FM_MAX_ROWS) return fm_why(w, FM_ERR_ARG, "%d rows, at most %d", *rows, FM_MAX_ROWS);
    return FM_OK;
}
inline int fm_check_dtype(FmWhy *w, int dtype) {
    return dtype == FM_DTYPE_F32 || dtype == FM_DTYPE_BF16 ? FM_OK : fm_why(w, FM_ERR_ARG, "dtype %d", dtype);
}
// a vector of rows: 16-byte aligned, its stride too, and at least a row wide
inline int fm_check_vec(FmWhy *w, const char *what, const void *p, int64_t stride, int64_t width, int dtype) {
    const int size = dtype == FM_DTYPE_BF16 ? 2 : 4;
    if (!p) return fm_why(w, FM_ERR_ARG, "null pointer: %s", what);
    if ((uintptr_t)p & 15) return fm_why(w, FM_ERR_ARG, "%s is not 16-byte aligned", what);
    if (stride < width) return fm_why(w, FM_ERR_ARG, "row stride %lld of %s below its width %lld", (long long)stride, what, (long long)width);
    if (stride > ((int64_t)1 << 40)) return fm_why(w, FM_ERR_ARG, "row stride %lld of %s", (long long)stride, what);
    if (stride * size % 16) return fm_why(w, FM_ERR_ARG, "row stride %lld of %s leaves rows unaligned (16 bytes)", (long long)stride, what);
    return FM_OK;
}
inline void fm_fill_seqs(FmSeqs *b, const int32_t *start, int n_seq) {
    memset(b, 0, sizeof *b);
    b->n_seq = n_seq;
    b->one_row = !start;
    if (start) memcpy(b->start, start, (size_t)(n_seq + 1) * sizeof(int));
}
inline int fm_gdn_check(FmWhy *w, const fm_gated_delta_args *p, FmGdn *a) {
    if (!p) return fm_why(w, FM_ERR_ARG, "null arguments");
    int rows, rc;
    if ((rc = fm_check_rows(w, p->seq_start, p->n_seq, &rows))) return rc;
    if ((rc = fm_check_dtype(w, p->dtype))) return rc;
    if (p->flags & ~FM_GDN_L2NORM) return fm_why(w, FM_ERR_ARG, "flags 0x%x", p->flags);
    if (p->k_heads < 1 || p->v_heads < p->k_heads || p->v_heads > 256 || p->v_heads % p->k_heads)
        return fm_why(w, FM_ERR_ARG, "%d key heads, %d value heads", p->k_heads, p->v_heads);
    if (p->k_dim != 64 && p->k_dim != 128) return fm_why(w, FM_ERR_UNSUPPORTED, "k_dim %d (64 or 128)", p->k_dim);
    if (p->v_dim < 16 || p->v_dim > 256 || p->v_dim % 16)
        return fm_why(w, FM_ERR_UNSUPPORTED, "v_dim %d (multiples of 16 up to 256)", p->v_dim);
    const int64_t kw = (int64_t)p->k_heads * p->k_dim, vw = (int64_t)p->v_heads * p->v_dim;
    if ((rc = fm_check_vec(w, "d_q", p->d_q, p->q_stride, kw, p->dtype))) return rc;
    if ((rc = fm_check_vec(w, "d_k", p->d_k, p->k_stride, kw, p->dtype))) return rc;
    if ((rc = fm_check_vec(w, "d_v", p->d_v, p->v_stride, vw, p->dtype))) return rc;
    if ((rc = fm_check_vec(w, "d_out", p->d_out, vw, vw, p->dtype))) return rc;
    if (!p->d_g || !p->d_beta || !p->d_state_out) return fm_why(w, FM_ERR_ARG, "null pointer");
    if (((uintptr_t)p->d_g | (uintptr_t)p->d_beta) & 3) return fm_why(w, FM_ERR_ARG, "d_g or d_beta not 4-byte aligned");
    const size_t state = (size_t)vw * p->k_dim * sizeof(float);
    // Outputs in address order: neighbours must lie a state apart, and an input may only meet the output
    // of its own sequence, exactly.
    std::pair<uintptr_t, int> outs[FM_MAX_SEQ];
    for (int i = 0; i < p->n_seq; i++) {
        const void *out = p->d_state_out[i], *in = p->d_state_in ? p->d_state_in[i] : nullptr;
        if (!out) return fm_why(w, FM_ERR_ARG, "null state output %d", i);
        if (((uintptr_t)out | (uintptr_t)in) & 15) return fm_why(w, FM_ERR_ARG, "state %d is not 16-byte aligned", i);
        outs[i] = {(uintptr_t)out, i};
    }
    std::sort(outs, outs + p->n_seq);
    for (int i = 1; i < p->n_seq; i++)
        if (outs[i].first - outs[i - 1].first < state)
            return fm_why(w, FM_ERR_ARG, "state outputs %d and %d overlap", outs[i - 1].second, outs[i].second);
    for (int i = 0; p->d_state_in && i < p->n_seq; i++) {
        const uintptr_t in = (uintptr_t)p->d_state_in[i];
        if (!in) continue;
        auto it = std::lower_bound(outs, outs + p->n_seq, std::make_pair(in, -1));
        if (it != outs + p->n_seq && it->first - in < state && !(it->first == in && it->second == i))
            return fm_why(w, FM_ERR_ARG, "state output %d overlaps state input %d", it->second, i);
        if (it != outs && in - (it - 1)->first < state)
            return fm_why(w, FM_ERR_ARG, "state output %d overlaps state input %d", (it - 1)->second, i);
    }
    a->k_heads = p->k_heads;
    a->v_heads = p->v_heads;
    a->k_dim = p->k_dim;
    a->v_dim = p->v_dim;
    a->l2norm = (p->flags & FM_GDN_L2NORM) != 0;
    a->scale = p->scale;
    a->q = p->d_q;
    a->k = p->d_k;
    a->v = p->d_v;
    a->q_stride = p->q_stride;
    a->k_stride = p->k_stride;
    a->v_stride = p->v_stride;
    a->g = p->d_g;
    a->beta = p->d_beta;
    a->out = p->d_out;
    return FM_OK;
}

inline int fm_kv_check(FmWhy *w, const fm_kv_cache *p, const int32_t *len, const int32_t *pages, int max_pages, FmKv *k) {
    if (!p->d_k || !p->d_v || !p->d_k_scale || !p->d_v_scale || !len || !pages)
        return fm_why(w, FM_ERR_ARG, "null pointer");
    if (((uintptr_t)p->d_k | (uintptr_t)p->d_v) & 15) return fm_why(w, FM_ERR_ARG, "cache codes are not 16-byte aligned");
    if (((uintptr_t)p->d_k_scale | (uintptr_t)p->d_v_scale | (uintptr_t)len | (uintptr_t)pages) & 3)
        return fm_why(w, FM_ERR_ARG, "scales, lengths or page table not 4-byte aligned");
    if (p->page_tokens != 16 && p->page_tokens != 32 && p->page_tokens != 64 && p->page_tokens != 128)
        return fm_why(w, FM_ERR_UNSUPPORTED, "pages of %d tokens (16, 32, 64 or 128)", p->page_tokens);
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
        return fm_why(w, FM_ERR_UNSUPPORTED, "head_dim %d (64, 128 or 256)", p->head_dim);
    if (p->n_pages < 1 || p->kv_heads < 1 || p->kv_heads > 256) return fm_why(w, FM_ERR_ARG, "%d pages, %d cache heads", p->n_pages, p->kv_heads);
    if (max_pages < 1 || (int64_t)max_pages * p->page_tokens > (int64_t)1 << 30)
        return fm_why(w, FM_ERR_ARG, "max_pages %d", max_pages);
    k->k = (int8_t *)p->d_k;
    k->v = (int8_t *)p->d_v;
    k->k_scale = p->d_k_scale;
    k->v_scale = p->d_v_scale;
    k->n_pages = p->n_pages;
    k->page_tokens = p->page_tokens;
    k->page_shift = __builtin_ctz((unsigned)p->page_tokens);
    k->kv_heads = p->kv_heads;
    k->len = len;
    k->pages = pages;
    k->max_pages = max_pages;
    return FM_OK;
}


// operands of fm_kv_append_dev / fm_kv_read_dev
inline int fm_kv_rows_check(FmWhy *w, const fm_kv_args *p, int read, FmKv *k, FmKvRows *x, FmSeqs *b) {
    if (!p) return fm_why(w, FM_ERR_ARG, "null arguments");
    int rows, rc;
    if ((rc = fm_check_rows(w, p->seq_start, p->n_seq, &rows))) return rc;
    if ((rc = fm_check_dtype(w, p->dtype))) return rc;
    if (read && p->dtype != FM_DTYPE_F32) return fm_why(w, FM_ERR_UNSUPPORTED, "rows are read back as fp32");
    if ((rc = fm_kv_check(w, &p->cache, p->d_len, p->d_pages, p->max_pages, k))) return rc;
    const int64_t width = (int64_t)p->cache.kv_heads * p->cache.head_dim;
    if ((rc = fm_check_vec(w, "d_k", p->d_k, p->k_stride, width, p->dtype))) return rc;
    if ((rc = fm_check_vec(w, "d_v", p->d_v, p->v_stride, width, p->dtype))) return rc;
    fm_fill_seqs(b, p->seq_start, p->n_seq);
    *x = FmKvRows{p->d_k, p->d_v, (float *)p->d_k, (float *)p->d_v, p->k_stride, p->v_stride};
    return FM_OK;
}

// ---- how a call is cut ---------------------------------------------------------------------
inline int fm_most_rows(const FmSeqs &b) {
    int most = b.one_row ? 1 : 0;
    if (!b.one_row)
        for (int i = 0; i < b.n_seq; i++) most = b.start[i + 1] - b.start[i] > most ? b.start[i + 1] - b.start[i] : most;
    return most;
}
inline int fm_all_rows(const FmSeqs &b) { return b.one_row ? b.n_seq : b.start[b.n_seq]; }

// Wide tiles: a workgroup takes whole tiles, or one of `splits` equal parts of a tile's steps where there are fewer
// tiles than workgroups.  Unit u of the launch is part u % splits of tile u / splits; tiles are numbered with the
// cache head running fastest (workgroups of one XCD then share a head's codes) and the sequences' last,
// longest tiles first.
struct FmWide {
    int first[FM_MAX_SEQ + 1];      // tiles of one head in the sequences before
};
inline void fm_attn_wide_tiles(const FmSeqs &b, int group, int wide, int narrow_most, FmWide *w) {
    w->first[0] = 0;
    for (int s = 0; s < b.n_seq; s++) w->first[s + 1] = w->first[s] + fm_attn_tiles(fm_seq_rows(b, s), group, wide, narrow_most);
}
struct FmWideUnit {
    int s, h, tile, part;
};
FM_HD FmWideUnit fm_attn_wide_unit(const FmWide &w, int n_seq, int kv_heads, int splits, int u) {
    FmWideUnit r;
    r.part = u % splits;
    u /= splits;
    r.h = u % kv_heads;
    const int t = w.first[n_seq] - 1 - u / kv_heads;
    int lo = 0, hi = n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (w.first[mid] <= t) lo = mid;
        else hi = mid;
    }
    r.s = lo;
    r.tile = t - w.first[lo];
    return r;
}
// Rounds of workgroups go through the units to and fro, so that whoever got the longest of a round gets
// the shortest of the next.
FM_HD int fm_attn_wide_pick(int round, int group, int groups) {
    return round * groups + (round & 1 ? groups - 1 - group : group);
}
// Parts of a tile: the number up to 16 whose rounds take least, a part costing a sixteenth of a tile's
// longest on top for being written and joined.
inline int fm_attn_splits(int64_t tiles, int groups, int most_steps) {
    int best = 1;
    double least = 1e30;
    for (int s = 1; s <= 16 && (s == 1 || s * FM_ATTN_WAVES <= most_steps); s++) {
        const double t = (double)((tiles * s + groups - 1) / groups) * (1.0 / s + (s > 1 ? 1.0 / 16 : 0.0));
        if (t < least * 0.999) least = t, best = s;
    }
    return best;
}

// Workgroups of a CU.  Narrow tiles: heads of 256 take a wave more registers than half a SIMD has (and a
// spilled one would wait for the codes in flight); heads of 128 have room for a second one (one bf16 row over
// 30000 keys 38.1 us with two, 38.6 with one; 32 rows over 8000 keys 38.1 / 37.2).
FM_HDC int fm_attn_per_cu(int D) { return D == 256 ? 1 : 2; }
// Columns of a sequence up to which it has narrow tiles: none where with wide tiles for all a workgroup would have
// FM_ATTN_MIXED_STEPS steps at most.
inline int fm_attn_narrow_most(const FmKv *c, const FmAttn *a, const FmSeqs *b, int n_cu) {
    if ((int64_t)fm_all_rows(*b) * a->group * c->kv_heads < FM_ATTN_WIDE_LEAST) return 0x7FFFFFFF;
    bool some = false;
    for (int s = 0; s < b->n_seq; s++) some |= fm_seq_rows(*b, s) * a->group > FM_ATTN_NARROW_MOST;
    if (!some || !a->wide_cols) return FM_ATTN_NARROW_MOST;
    FmWide w;
    fm_attn_wide_tiles(*b, a->group, a->wide_cols, 0, &w);
    const int64_t tiles = (int64_t)w.first[b->n_seq] * c->kv_heads;
    const int steps = (a->max_len + FM_ATTN_KEYS - 1) / FM_ATTN_KEYS, splits = fm_attn_splits(tiles, n_cu, steps);
    const int64_t of_one = (tiles * splits + n_cu - 1) / n_cu * ((steps + splits - 1) / splits);
    return of_one <= FM_ATTN_MIXED_STEPS ? 0 : FM_ATTN_NARROW_MOST;
}

// Steps of the narrow launch's tiles if every sequence is max_len long.
inline int64_t fm_attn_most_steps(const FmKv &c, const FmAttn &a, const FmSeqs &b) {
    int64_t most = 0;
    for (int s = 0; s < b.n_seq; s++)
        most += (int64_t)c.kv_heads * fm_attn_tiles(fm_seq_rows(b, s), a.group, 0, a.narrow_most) * ((a.max_len + FM_ATTN_KEYS - 1) / FM_ATTN_KEYS + 1);
    return most;
}
// Attention: the workgroups that fit on the chip share the steps, fewer if there cannot be as many.  Sets
// n_tiles (0: no sequence for this launch), groups and splits; returns the workspace: of narrow tiles two parts
// per workgroup and the steps before each sequence, of wide ones the parts of split tiles.
inline size_t fm_attn_plan(const FmKv *c, FmAttn *a, const FmSeqs *b, int D, int n_cu, int wide) {
    const int64_t have = (int64_t)c->max_pages * c->page_tokens;
    if (a->max_len > have) a->max_len = (int)have;
    a->wide = wide;
    a->narrow_most = fm_attn_narrow_most(c, a, b, n_cu);
    a->n_tiles = 0;
    a->splits = 1;
    for (int s = 0; s < b->n_seq; s++) a->n_tiles = std::max(a->n_tiles, fm_attn_tiles(fm_seq_rows(*b, s), a->group, wide, a->narrow_most));
    if (!a->n_tiles) return 0;
    if (wide) {
        FmWide w;
        fm_attn_wide_tiles(*b, a->group, wide, a->narrow_most, &w);
        const int64_t tiles = (int64_t)w.first[b->n_seq] * c->kv_heads;
        a->splits = fm_attn_splits(tiles, n_cu, (a->max_len + FM_ATTN_KEYS - 1) / FM_ATTN_KEYS);
        a->groups = (int)(tiles * a->splits < n_cu ? tiles * a->splits : n_cu);
        return a->splits == 1 ? 0 : (size_t)tiles * a->splits * wide * (D + 2) * sizeof(float);
    }
    const int64_t groups = (fm_attn_most_steps(*c, *a, *b) + FM_ATTN_WAVES - 1) / FM_ATTN_WAVES, fit = fm_attn_per_cu(D) * n_cu;
    a->groups = (int)(groups < 1 ? 1 : groups > fit ? fit : groups);
    return (size_t)2 * a->groups * fm_attn_cols(wide) * (D + 2) * sizeof(float) + (FM_MAX_SEQ + 1) * sizeof(int);
}

inline int fm_attn_check(FmWhy *w, const fm_attn_args *p, int n_cu, FmKv *k, FmAttn *a, FmSeqs *b, size_t *ws) {
    if (!p) return fm_why(w, FM_ERR_ARG, "null arguments");
    int rows, rc;
    if ((rc = fm_check_rows(w, p->seq_start, p->n_seq, &rows))) return rc;
    if ((rc = fm_check_dtype(w, p->dtype))) return rc;
    if ((rc = fm_kv_check(w, &p->cache, p->d_len, p->d_pages, p->max_pages, k))) return rc;
    if (p->q_heads < 1 || p->q_heads > 1024 || p->q_heads % p->cache.kv_heads)
        return fm_why(w, FM_ERR_ARG, "%d query heads on %d cache heads", p->q_heads, p->cache.kv_heads);
    if (p->max_len < 0) return fm_why(w, FM_ERR_ARG, "max_len %d", p->max_len);
    const int64_t width = (int64_t)p->q_heads * p->cache.head_dim;
    if ((rc = fm_check_vec(w, "d_q", p->d_q, p->q_stride, width, p->dtype))) return rc;
    if ((rc = fm_check_vec(w, "d_out", p->d_out, width, width, p->dtype))) return rc;
    memset(a, 0, sizeof *a);
    a->q = p->d_q;
    a->q_stride = p->q_stride;
    a->out = p->d_out;
    a->q_heads = p->q_heads;
    a->group = p->q_heads / p->cache.kv_heads;
    a->scale_log2 = (float)((double)p->scale * 1.4426950408889634);
    a->max_len = p->max_len;
    a->wide_cols = fm_attn_wide_cols(p->dtype == FM_DTYPE_BF16);
    fm_fill_seqs(b, p->seq_start, p->n_seq);
    FmAttn other = *a;       // (the two launches run one after the other in the same workspace)
    const size_t wide = fm_attn_plan(k, &other, b, p->cache.head_dim, n_cu, a->wide_cols);
    *ws = fm_attn_plan(k, a, b, p->cache.head_dim, n_cu, 0);
    if (wide > *ws) *ws = wide;
    // (the device numbers the steps it finds in 32 bits)
    const int64_t most = fm_attn_most_steps(*k, *a, *b);
    if (most > FM_ATTN_MOST_STEPS)
        return fm_why(w, FM_ERR_ARG, "%lld steps of %d keys at max_len, at most %d", (long long)most, FM_ATTN_KEYS, FM_ATTN_MOST_STEPS);
    return FM_OK;
}

inline int fm_logprob_check(FmWhy *w, int rows, int vocab, int top_n) {
    if (rows < 1 || rows > FM_MAX_ROWS) return fm_why(w, FM_ERR_ARG, "%d rows outside 1..%d", rows, FM_MAX_ROWS);
    if (vocab < 1 || vocab > (1 << 24)) return fm_why(w, FM_ERR_ARG, "vocab %d", vocab);
    if (top_n < 0 || top_n > 32 || top_n > vocab) return fm_why(w, FM_ERR_ARG, "top_n %d outside 0..min(32, vocab)", top_n);
    return FM_OK;
}

inline int fm_logprob_args_check(FmWhy *w, const void *d_logits, int rows, int vocab, int64_t row_stride, const void *d_tokens,
                                 int top_n, const void *d_logprob, const void *d_entropy, const void *d_top_ids,
                                 const void *d_top_logprobs) {
    if (!d_logits) return fm_why(w, FM_ERR_ARG, "null pointer");
    int rc = fm_logprob_check(w, rows, vocab, top_n);
    if (rc) return rc;
    if (row_stride < vocab || row_stride > ((int64_t)1 << 40))
        return fm_why(w, FM_ERR_ARG, "row stride %lld, vocab %d", (long long)row_stride, vocab);
    if (!d_tokens != !d_logprob) return fm_why(w, FM_ERR_ARG, "tokens and their log probabilities go together");
    if (!d_top_ids != !d_top_logprobs || !d_top_ids != !top_n)
        return fm_why(w, FM_ERR_ARG, "top_n, top ids and top log probabilities go together");
    if (((uintptr_t)d_logits | (uintptr_t)d_tokens | (uintptr_t)d_logprob | (uintptr_t)d_entropy | (uintptr_t)d_top_ids |
         (uintptr_t)d_top_logprobs) & 3)
        return fm_why(w, FM_ERR_ARG, "pointer not 4-byte aligned");
    return FM_OK;
}
