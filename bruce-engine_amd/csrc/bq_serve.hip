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

size_t bq_attn_shared_workspace_bytes(int n_seq, int rows, int q_heads, int kv_heads, int head_dim, int max_len, int n_groups, int max_prefix) {
    if (n_seq <= 0 || n_seq > 65535 || rows < 1 || rows > BQ_MAX_ROWS || kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads <= 0 ||
        head_dim <= 0 || max_len < 0 || n_groups < 1 || max_prefix < 0 || device_ready() != BQ_OK)
        return 0;
    // of either type and any window: the pieces are the most without one
    max_prefix = std::min(max_prefix, max_len);
    size_t most = 0;
    for (int type : {kKvBf16, kKvQ8})
        most = std::max(most, shared_part_floats(shared_plan(type, n_seq, rows, q_heads, kv_heads, head_dim, max_len, n_groups, max_prefix, 0, 0,
                                                             device_cus()), n_seq * rows, q_heads, head_dim));
    return most * sizeof(float);
}

int bq_attn_decode_shared(const bq_kv_cache* c, const bq_attn_args* args, const bq_attn_prefix* prefix, bq_stream_t st) {
    if (int r = device_ready()) return r;
    KvView kv;
    int type;
    if (int r = view_of(c, kv, type)) return r;
    if (!args || !prefix) return BQ_EINVAL;
    bq_attn_args a = *args;
    bq_attn_prefix x = *prefix;
    if (int r = attn_check(kv, a)) return r;
    if (a.row0 || (int64_t)kv.n_seq * a.rows != a.n_rows) return BQ_EINVAL;
    if (!x.group0 || !x.len || x.n_groups < 1 || x.max_len < 0) return BQ_EINVAL;
    if (a.rows > BQ_MAX_ROWS) return BQ_UNSUPPORTED;
    x.max_len = std::min(x.max_len, a.max_len);
    const SharedPlan s = shared_plan(type, kv.n_seq, a.rows, a.q_heads, kv.heads, kv.D, a.max_len, x.n_groups, x.max_len, a.window, a.sinks,
                                     device_cus());
    // a grid has at most 2^32 - 1 lanes, 256 a workgroup: of all pieces, and of all rows
    constexpr int64_t kGroups = (1 << 24) - 1;
    if (s.punits + (int64_t)kv.n_seq * s.ttiles * kv.heads * s.tsplit > kGroups || (int64_t)a.n_rows * a.q_heads > kGroups) return BQ_UNSUPPORTED;
    if (!a.work || !al16(a.work) || a.work_bytes < shared_part_floats(s, a.n_rows, a.q_heads, kv.D) * sizeof(float)) return BQ_EINVAL;
    return from_hip(launch_attn_shared(kv, type, a, x, s, (hipStream_t)st));
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
        if (r == BQ_OK && b.attn && b.shared)
            r = b.prefill ? BQ_EINVAL : bq_attn_decode_shared(b.kv, b.attn, b.shared, st);
        else if (r == BQ_OK && b.attn)
            r = b.prefill ? bq_attn_prefill(b.kv, b.attn, st) : bq_attn_decode(b.kv, b.attn, st);
    }
    if (p->status == BQ_OK) p->status = r;
}

size_t bq_lora_workspace_bytes(int rows, int rank, int n_parts) {
    return rows > 0 && rank > 0 && rank <= BQ_MAX_RANK && n_parts > 0 && n_parts <= BQ_MAX_PARTS ? lora_work_bytes(rows, rank, n_parts) : 0;
}

int bq_lora(const bq_lora_args* a, bq_stream_t st) {
    if (int r = device_ready()) return r;
    if (!a || a->rows < 0 || a->K <= 0 || a->rank <= 0 || a->n_adapters <= 0 || a->n_parts < 1 || a->n_parts > BQ_MAX_PARTS) return BQ_EINVAL;
    if (a->x_type != BQ_TYPE_Q8_0 && !float_type(a->x_type)) return BQ_EINVAL;
    if (a->K % 32 || a->rank % 8 || a->rank > BQ_MAX_RANK) return BQ_UNSUPPORTED;
    int64_t outputs = 0;
    for (int i = 0; i < a->n_parts; ++i) {
        const bq_lora_part& p = a->parts[i];
        if (p.N <= 0) return BQ_EINVAL;
        if (p.N % 16) return BQ_UNSUPPORTED;
        outputs += (p.N + 255) / 256;
    }
    // grid dimensions: outputs and rows of one launch
    if (outputs > 65535 || a->rows > BQ_MAX_LORA_ROWS) return BQ_UNSUPPORTED;
    if (a->rows == 0) return BQ_OK;
    if (!a->x || !al16(a->x) || !a->adapter) return BQ_EINVAL;
    if (a->x_type == BQ_TYPE_Q8_0 ? !a->xd : a->ldx < a->K || a->ldx % (a->x_type == BQ_TYPE_F32 ? 4 : 8)) return BQ_EINVAL;
    for (int i = 0; i < a->n_parts; ++i) {
        const bq_lora_part& p = a->parts[i];
        if (!p.a || !p.b || !p.y || !al16(p.a) || !al16(p.b) || !al16(p.y) || !al16(p.base) || p.ldy < p.N || (p.ldy & 3)) return BQ_EINVAL;
        for (int j = 0; j < a->n_parts; ++j)  // the parts run side by side
            if (j != i && (a->parts[j].y == p.y || a->parts[j].y == p.base)) return BQ_EINVAL;
        if (p.base && (p.ldbase < p.N || (p.ldbase & 3) || (p.base == p.y && p.ldbase != p.ldy))) return BQ_EINVAL;
    }
    if (!a->work || !al16(a->work) || a->work_bytes < lora_work_bytes(a->rows, a->rank, a->n_parts)) return BQ_EINVAL;
    return from_hip(launch_lora(*a, (hipStream_t)st));
}

void bq_lora_hook(void* user, int block, int proj, bq_stream_t st) {
    bq_lora_plan* p = (bq_lora_plan*)user;
    if (!p) return;
    int r = BQ_OK;
    if (block < 0 || block >= p->n_blocks || !p->blocks || proj < 0 || proj >= BQ_N_PROJ)
        r = BQ_EINVAL;
    else if (const bq_lora_args* a = p->blocks[block].proj[proj])
        r = bq_lora(a, st);
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

size_t bq_logprobs_workspace_bytes(int rows, int vocab, int top) {
    return rows > 0 && vocab > 0 && vocab <= (1 << 20) && top >= 0 && top <= BQ_MAX_TOP ? logprob_work_bytes(rows, vocab, top) : 0;
}

int bq_logprobs(const bq_logprobs_args* a, bq_stream_t st) {
    if (int r = device_ready()) return r;
    if (!a || a->rows < 0 || a->vocab <= 0 || a->ld < a->vocab || a->top < 0) return BQ_EINVAL;
    if (a->vocab > (1 << 20) || a->rows > 65535 || a->top > BQ_MAX_TOP) return BQ_UNSUPPORTED;
    // what a result is of, or where it goes
    if (!a->tokens && (a->logprob || a->rank)) return BQ_EINVAL;
    if (!a->logprob && !a->rank && !a->entropy && !(a->top && (a->top_tokens || a->top_logprobs))) return BQ_EINVAL;
    if (a->rows == 0) return BQ_OK;
    if (!a->logits || ((uintptr_t)a->logits & 3) || !a->work || !al16(a->work) || a->work_bytes < logprob_work_bytes(a->rows, a->vocab, a->top))
        return BQ_EINVAL;
    return from_hip(launch_logprobs(*a, (hipStream_t)st));
}

}  // extern "C"
