// bq_serve.hip -- C ABI of the serving operators (include/bq.h): the paged
// cache, attention over it, sampling, and the decode step's attention hook.
// Argument checks and dispatch; nothing here allocates or synchronises.
#include <algorithm>
#include <cmath>

#include "../../include/bq.h"
#include "bq_internal.hpp"
#include "bq_kv.hpp"

using namespace bq;

namespace {

bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }
int from_hip(hipError_t e) { return e == hipSuccess ? BQ_OK : -(int)e; }

bool layout_ok(int type, int kv_heads, int D, int P) {
    return (type == BQ_TYPE_BF16 || type == BQ_TYPE_Q8_0) && kv_heads > 0 && kv_heads <= 65535 &&
           (D == 64 || D == 128 || D == 256) && (P == 16 || P == 32 || P == 64 || P == 128 || P == 256);
}
int head_bytes(int type, int D, int P) { return type == BQ_TYPE_BF16 ? 4 * P * D : 2 * P * D + P * D / 8; }
bool float_type(int t) { return t == BQ_TYPE_F32 || t == BQ_TYPE_BF16; }

// BQ_OK and the device view, or the code to return
int view_of(const bq_kv_cache* c, KvView& v, int& type) {
    if (!c || !c->pages || !c->table || !al16(c->pages) || c->n_pages <= 0 || c->n_seq <= 0 || c->max_pages <= 0) return BQ_EINVAL;
    if (!layout_ok(c->type, c->kv_heads, c->head_dim, c->page_tokens) || c->n_seq > 65535) return BQ_UNSUPPORTED;
    v.pages = (char*)c->pages;
    v.table = c->table;
    v.head_bytes = head_bytes(c->type, c->head_dim, c->page_tokens);
    v.page_bytes = (int64_t)v.head_bytes * c->kv_heads;
    v.heads = c->kv_heads;
    v.D = c->head_dim;
    v.P = c->page_tokens;
    v.plog = __builtin_ctz((unsigned)c->page_tokens);
    v.n_pages = c->n_pages;
    v.n_seq = c->n_seq;
    // token indices are 32-bit, and a tile's end is one past its last token: room for
    // one tile (and the tokens of a window's last step) above the longest sequence
    if (c->max_pages > ((INT32_MAX - 127) >> v.plog)) return BQ_UNSUPPORTED;
    v.max_pages = c->max_pages;
    type = c->type == BQ_TYPE_BF16 ? kKvBf16 : kKvQ8;
    return BQ_OK;
}

int attn_check(const KvView& kv, bq_attn_args& a) {
    if (!a.q || !a.out || !a.kv_len || !al16(a.q) || !al16(a.out) || !float_type(a.q_type) || !float_type(a.out_type)) return BQ_EINVAL;
    if (a.q_heads <= 0 || a.rows <= 0 || a.n_rows < 0 || a.max_len < 0 || a.window < 0 || a.sinks < 0 || !(a.scale > 0.f) ||
        !std::isfinite(a.scale))
        return BQ_EINVAL;
    const int64_t width = (int64_t)a.q_heads * kv.D;
    if (a.ldq < width || a.ldo < width || (a.ldq & 7) || (a.ldo & 7)) return BQ_EINVAL;
    if (a.q_heads % kv.heads != 0 || a.q_heads / kv.heads > 64) return BQ_UNSUPPORTED;
    a.max_len = (int)std::min<int64_t>(a.max_len, (int64_t)kv.max_pages * kv.P);
    // a window that no position reaches past is none; sinks count up to the length
    if (a.window >= a.max_len) a.window = 0;
    a.sinks = a.window ? std::min(a.sinks, a.max_len) : 0;
    return BQ_OK;
}

}  // namespace

extern "C" {

size_t bq_kv_page_bytes(int type, int kv_heads, int head_dim, int page_tokens) {
    if (!layout_ok(type, kv_heads, head_dim, page_tokens)) return 0;
    return (size_t)head_bytes(type, head_dim, page_tokens) * kv_heads;
}

int bq_append(const bq_kv_cache* c, const bq_append_args* a, bq_stream_t st) {
    if (int r = device_ready()) return r;
    KvView kv;
    int type;
    if (int r = view_of(c, kv, type)) return r;
    if (!a || a->rows < 0 || a->q_heads <= 0 || a->q_heads > 65535 || !float_type(a->q_type) || a->n_pos < 0) return BQ_EINVAL;
    if (a->rows == 0) return BQ_OK;
    if (!a->q || !a->k || !a->v || !a->pos || !a->q_out) return BQ_EINVAL;
    if (!al16(a->q) || !al16(a->k) || !al16(a->v) || !al16(a->q_out) || !al16(a->q_weight) || !al16(a->k_weight) || !al16(a->rope))
        return BQ_EINVAL;
    const int64_t qw = (int64_t)a->q_heads * kv.D, kw = (int64_t)kv.heads * kv.D;
    if (a->ldq < qw || a->ldk < kw || a->ldv < kw || ((a->ldq | a->ldk | a->ldv) & 3)) return BQ_EINVAL;
    if (a->rot < 0 || a->rot > kv.D || (a->rot & 7) || (a->rot > 0 && !a->rope)) return BQ_EINVAL;
    // queries in place: a lane writes what it read, where the rows lie alike
    if (a->q_out == (const void*)a->q && (a->q_type != BQ_TYPE_F32 || a->ldq != qw)) return BQ_EINVAL;
    return from_hip(launch_append(kv, type, *a, (hipStream_t)st));
}

int bq_kv_read(const bq_kv_cache* c, const int32_t* seq, const int32_t* pos, int rows, uint16_t* k, uint16_t* v, bq_stream_t st) {
    if (int r = device_ready()) return r;
    KvView kv;
    int type;
    if (int r = view_of(c, kv, type)) return r;
    if (rows < 0) return BQ_EINVAL;
    if (rows == 0 || (!k && !v)) return BQ_OK;
    if (!pos || !al16(k) || !al16(v)) return BQ_EINVAL;
    return from_hip(launch_kv_read(kv, type, seq, pos, rows, k, v, (hipStream_t)st));
}

size_t bq_attn_workspace_bytes(int n_seq, int rows, int q_heads, int kv_heads, int head_dim, int max_len) {
    if (n_seq <= 0 || rows < 1 || rows > BQ_MAX_ROWS || kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads <= 0 || head_dim <= 0 ||
        max_len < 0 || device_ready() != BQ_OK)
        return 0;
    // of either type: a q8 cache's tokens are cut earlier
    const int n = decode_splits(kKvQ8, n_seq, rows, q_heads, kv_heads, head_dim, max_len, device_cus());
    return n > 1 ? n * decode_part_floats(n_seq, rows, q_heads, kv_heads, head_dim) * sizeof(float) : 0;
}

size_t bq_attn_prefill_workspace_bytes(int type, int n_seq, int rows, int n_rows, int q_heads, int kv_heads, int head_dim, int max_len) {
    if (n_seq <= 0 || rows < 1 || n_rows < 1 || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads != 0 || head_dim <= 0 ||
        max_len < 0 || device_ready() != BQ_OK)
        return 0;
    const int n = prefill_splits(n_seq, std::min(rows, n_rows), q_heads, kv_heads, head_dim, max_len, device_cus());
    const size_t parts = n > 1 ? n * prefill_part_floats(n_rows, q_heads, head_dim) * sizeof(float) : 0;
    return parts + prefill_stage_bytes(type == BQ_TYPE_Q8_0 ? kKvQ8 : kKvBf16, n_seq, std::min(rows, n_rows), q_heads, kv_heads,
                                       head_dim, max_len);
}

int bq_attn_decode(const bq_kv_cache* c, const bq_attn_args* args, bq_stream_t st) {
    if (int r = device_ready()) return r;
    KvView kv;
    int type;
    if (int r = view_of(c, kv, type)) return r;
    if (!args) return BQ_EINVAL;
    bq_attn_args a = *args;
    if (int r = attn_check(kv, a)) return r;
    if (a.row0 || (int64_t)kv.n_seq * a.rows != a.n_rows) return BQ_EINVAL;
    if (a.rows > BQ_MAX_ROWS) return BQ_UNSUPPORTED;
    if (!al16(a.work) || (a.work_bytes && !a.work)) return BQ_EINVAL;
    int n = decode_splits(type, kv.n_seq, a.rows, a.q_heads, kv.heads, kv.D, decode_reach(a.rows, a.window, a.sinks, a.max_len), device_cus());
    const size_t part = decode_part_floats(kv.n_seq, a.rows, a.q_heads, kv.heads, kv.D) * sizeof(float);
    n = (int)std::min<size_t>(n, std::max<size_t>(1, a.work_bytes / part));
    return from_hip(launch_attn_decode(kv, type, a, n, (hipStream_t)st));
}

int bq_attn_prefill(const bq_kv_cache* c, const bq_attn_args* args, bq_stream_t st) {
    if (int r = device_ready()) return r;
    KvView kv;
    int type;
    if (int r = view_of(c, kv, type)) return r;
    if (!args) return BQ_EINVAL;
    bq_attn_args a = *args;
    if (int r = attn_check(kv, a)) return r;
    if (!a.row0 && (kv.n_seq != 1 || a.rows != a.n_rows)) return BQ_EINVAL;
    if (a.n_rows == 0) return BQ_OK;
    if ((int64_t)a.rows * (a.q_heads / kv.heads) > INT32_MAX / 2) return BQ_UNSUPPORTED;
    if (!al16(a.work) || (a.work_bytes && !a.work)) return BQ_EINVAL;
    // the converted tiles first, the pieces in what is left
    size_t stage = prefill_stage_bytes(type, kv.n_seq, std::min(a.rows, a.n_rows), a.q_heads, kv.heads, kv.D, a.max_len);
    if (stage > a.work_bytes) stage = 0;
    int n = prefill_splits(kv.n_seq, std::min(a.rows, a.n_rows), a.q_heads, kv.heads, kv.D, prefill_reach(a.window, a.sinks, a.max_len), device_cus());
    const size_t part = prefill_part_floats(a.n_rows, a.q_heads, kv.D) * sizeof(float);
    n = (int)std::min<size_t>(n, std::max<size_t>(1, (a.work_bytes - stage) / part));
    // (sequence, piece) is one grid dimension
    n = std::max(1, std::min(n, 65535 / kv.n_seq));
    return from_hip(launch_attn_prefill(kv, type, a, stage, n, device_cus(), (hipStream_t)st));
}

void bq_attn_hook(void* user, int block, bq_stream_t st) {
    bq_attn_plan* p = (bq_attn_plan*)user;
    if (!p) return;
    int r = BQ_OK;
    if (block < 0 || block >= p->n_blocks || !p->blocks) {
        r = BQ_EINVAL;
    } else if (p->blocks[block].kv) {
        const bq_attn_block& b = p->blocks[block];
        if (b.append) r = bq_append(b.kv, b.append, st);
        if (r == BQ_OK && b.attn) r = b.prefill ? bq_attn_prefill(b.kv, b.attn, st) : bq_attn_decode(b.kv, b.attn, st);
    }
    if (p->status == BQ_OK) p->status = r;
}

size_t bq_sample_workspace_bytes(int rows, int vocab) {
    return rows > 0 && vocab > 0 && vocab <= (1 << 20) ? sample_work_bytes(rows, vocab) : 0;
}

int bq_sample(const float* logits, int64_t ld, int rows, int vocab, const float* temperature, const int32_t* top_k, const float* top_p,
              const float* min_p, const float* u, int32_t* out, void* work, size_t work_bytes, bq_stream_t st) {
    if (int r = device_ready()) return r;
    if (rows < 0 || vocab <= 0 || ld < vocab) return BQ_EINVAL;
    if (vocab > (1 << 20) || rows > 65535) return BQ_UNSUPPORTED;
    if (rows == 0) return BQ_OK;
    if (!logits || !u || !out || !work || ((uintptr_t)logits & 3) || !al16(work) || work_bytes < sample_work_bytes(rows, vocab)) return BQ_EINVAL;
    return from_hip(launch_sample(logits, ld, rows, vocab, temperature, top_k, top_p, min_p, u, out, work, (hipStream_t)st));
}

}  // extern "C"
