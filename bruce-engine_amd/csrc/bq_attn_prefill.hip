// bq_attn_prefill.hip -- attention of prompt chunks over the paged cache.
//
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q.k_j
// in one pass over 64-token tiles with a running m.  4 D flops per visible
// (row, token) pair and head: the matrix pipe bounds it.
//
// A workgroup takes 128 query rows of one key-value head (the group's heads
// times the chunk's rows, heads fastest), four waves of 32 rows.  Scores are
// computed transposed, S^T = K Q^T on 32x32x16 MFMA, so a lane holds tokens of
// one query row: the softmax needs one exchange between the wave's halves, and
// only when the maximum moves.  The K tile's rows are dealt so that a lane
// ends with runs of 8 tokens, the B operand of O^T = V^T P^T: the weights
// stay in their lane, rounded to bf16 (at most 2^-8 of a weight, as the queries are;
// sums and statistics are fp32).  K and V are in the A operands' order in the
// cache already, so a tile is copied to LDS as it lies (direct to LDS for
// bf16; q8 is dequantized on the way) while the one before is computed.
// Over a q8 cache the score product is fp16: a code times its scale and an
// fp32 query need more than bf16's 8 bits (rounding both to bf16 moves an
// output by 0.5% of its length at scores of a few units, fp16 by what the
// weights' rounding does); each token and each query row is divided by a power
// of two first, which keeps fp32's range.  Where the q8 tiles are converted ahead
// of the attention (k_stage_q8), values and weights are fp16 too, 2^-11 of each
// instead of 2^-8, for 4% of the time; a tile's values then stand over a power of
// two that brings its largest scale into fp16's range, taken from the tokens that
// some row sees.
//
// Few rows over many tokens are split over workgroups (prefill_splits) and joined
// in the pieces' order; a short chunk halves the row tiles (half_tiles).
// Measured (32 heads of 128 over 4, bf16): 8192 rows 555 us, 990 TFLOP/s of the
// 1187 that a large library product reaches; 512 rows 15.4 us, where the launch,
// the first tile's latency (page, then K and V) and the epilogue are most of it.
// Five ragged chunks of up to 700 rows over a q8 cache, window 2048: 175 us for
// 77.7 GFLOP; the 584 row tiles fill 512 slots once and then 72 of them again.
#include <algorithm>

#include "bq_internal.hpp"
#include "bq_kv.hpp"

namespace bq {

namespace {
constexpr int kBN = 64;          // tokens of a tile
// a q8 cache's tiles turned into the products' operands ahead of the attention:
// fp16 keys and values as they lie in LDS, what the tokens' scores are
// multiplied by, the mask of unmapped tokens, the power of two of the values
constexpr int kKvStaged = 2;
constexpr int64_t tile_record(int D) { return 4 * kBN * D + 512; }
constexpr int kPiece = 8;        // tiles of a piece at least, where the tokens are split
constexpr float kNone = -1e30f;  // the running maximum before any token
constexpr float kLazy = 8.f;     // it moves when a score passes it by more (log2)

struct PrefillP {
    KvView kv;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    const int32_t* row0;
    const int32_t* kv_len;
    float* part;  // nsplit > 1: [nsplit][n_rows][q_heads][D], then [..][2] (m, l)
    int64_t ml;   // floats before the (m, l) part
    char* stage;  // kKvStaged: [n_seq][heads][stage_tiles] records of a tile
    int stage_tiles;
    int G, q_heads, n_rows, max_rows, max_len, window, sinks, q_bf16, out_bf16, nsplit;
    float scale;  // scale * log2(e)
};

// a sequence's rows of q and out, kept inside the buffers whatever row0 holds
BQ_DEV void rows_of(const PrefillP& p, int seq, int& base, int& rows) {
    const int b0 = p.row0 ? p.row0[seq] : 0, b1 = p.row0 ? p.row0[seq + 1] : p.n_rows;
    base = min(max(b0, 0), p.n_rows);
    rows = min(min(max(b1, 0), p.n_rows) - base, p.max_rows);
}

BQ_DEV f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

BQ_DEV f32x16 mfma32h(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// 16 bytes per lane straight to LDS at lds + 16 * lane (m0: see bq_gemm.hip's
// dma16), from a lane's own address or from a wave's base + 16 * lane
BQ_DEV void copy_lds(const void* src, const void* lds) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(m0) : "m0", "memory");
}
BQ_DEV void copy_lds_row(const void* base, uint32_t off, const void* lds) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(m0) : "m0", "memory");
}

// four int8 codes times their scales -> bf16
BQ_DEV u32x2 dequant4(uint32_t w, float a, float b, float c, float d) {
    return u32x2{f2bf2((float)(int8_t)w * a, (float)(int8_t)(w >> 8) * b),
                 f2bf2((float)(int8_t)(w >> 16) * c, (float)((int32_t)w >> 24) * d)};
}
// four int8 codes times one fp16 scale
BQ_DEV u32x2 dequant4h(uint32_t w, f16x2 scale) {
    f16x2 lo, hi;
    codes_f16(w, lo, hi);
    return u32x2{__builtin_bit_cast(uint32_t, lo * scale), __builtin_bit_cast(uint32_t, hi * scale)};
}

// four values of a row (zeros where the row saw nothing: l is 0)
BQ_DEV void store4(const PrefillP& p, size_t at, f32x4 y, float l) {
    if (l == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
    if (p.out_bf16)
        *(u32x2*)((uint16_t*)p.out + at) = u32x2{f2bf2(y[0], y[1]), f2bf2(y[2], y[3])};
    else
        *(f32x4*)((float*)p.out + at) = y;
}

// 2^e of a q8 token's largest key scale, from its bf16 bits
BQ_DEV int key_power(uint32_t top) { return max(-100, min(100, (int)(top >> 7) - 127)); }
// 16 key codes (dims 64c + 8g.. and 64c + 32 + 8g..) times two scales over the token's power of two
BQ_DEV u32x4 half_keys(u32x4 codes, int k, uint16_t scale, float down) {
    const _Float16 sh = (_Float16)(bf2f(scale) * down);
    const u32x2 a = dequant4h(codes[2 * k], f16x2{sh, sh}), b = dequant4h(codes[2 * k + 1], f16x2{sh, sh});
    return u32x4{a[0], a[1], b[0], b[1]};
}
// 8 tokens' codes of a value's dim times their scales
BQ_DEV u32x4 bf16_values(u32x4 codes, int k, u32x4 scales) {
    float y[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) y[x] = as_float(x & 1 ? scales[x >> 1] & 0xFFFF0000u : scales[x >> 1] << 16);
    const u32x2 a = dequant4(codes[2 * k], y[0], y[1], y[2], y[3]), b = dequant4(codes[2 * k + 1], y[4], y[5], y[6], y[7]);
    return u32x4{a[0], a[1], b[0], b[1]};
}
// 2^e of a tile's values from its largest value scale: 0 where fp16 holds the
// codes times their scales as they are, else what brings the scale into 2^-8 .. 2^9
BQ_DEV int value_power(uint32_t top) {
    const int e = (int)(top >> 7) - 127;
    return top == 0 ? -100 : e > 8 ? min(100, e - 8) : e < -8 ? max(-100, e + 8) : 0;
}
// a wave's largest, or another whose value_power is the same
BQ_DEV uint32_t wave_top(uint32_t top) {
    if (__any(value_power(top) == 0) && !__any(value_power(top) > 0)) return 0x3F80;
    for (int d = 1; d < 64; d <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d, 64));
    return top;
}
// 8 tokens' codes of a value's dim times their scales, over the tile's power of two
BQ_DEV u32x4 half_values(u32x4 codes, int k, u32x4 scales, float down) {
    f16x2 lo, hi;
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        codes_f16(codes[2 * k + w], lo, hi);
        const uint32_t a = scales[2 * w], b = scales[2 * w + 1];
        r[2 * w] = __builtin_bit_cast(uint32_t, lo * f16x2{(_Float16)(as_float(a << 16) * down), (_Float16)(as_float(a & 0xFFFF0000u) * down)});
        r[2 * w + 1] = __builtin_bit_cast(uint32_t, hi * f16x2{(_Float16)(as_float(b << 16) * down), (_Float16)(as_float(b & 0xFFFF0000u) * down)});
    }
    return r;
}

// One 64-token tile of one head into its record.  Every row tile of a prompt
// reads the tile again: converting it there each time costs as many vector
// instructions as the softmax, so it is done once, in a launch of its own, where
// there are enough row tiles (kStageRows).
template <int D>
__global__ void __launch_bounds__(256) k_stage_q8(PrefillP p) {
    const KvView& kv = p.kv;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, tile = blockIdx.x, h = blockIdx.y, seq = blockIdx.z, P = kv.P;
    int base, rows;
    rows_of(p, seq, base, rows);
    const int len = min(max(p.kv_len[seq], 0), min(p.max_len, kv.max_pages << kv.plog));
    const int t0 = tile * kBN;
    if (rows <= 0 || t0 >= len) return;
    if (p.window && t0 + kBN <= len - rows - p.window + 1 && t0 >= p.sinks) return;  // no row sees it
    char* rec = p.stage + (((size_t)seq * kv.heads + h) * p.stage_tiles + tile) * tile_record(D);
    const int pid = t0 + lane < len ? kv_page(kv, seq, t0 + lane) : -1, tk = (t0 + lane) & (P - 1);
    const char* head = kv.pages + (size_t)h * kv.head_bytes;
    const char* kb = head + (int64_t)max(pid, 0) * kv.page_bytes;
    uint16_t ks[D / 32];
    uint32_t top = 0, vtop = 0;  // the token's largest key and value scale
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
        ks[e] = *(const uint16_t*)(kb + kv_ks_off(P, D, e, tk));
        top = max(top, (uint32_t)ks[e]);
        vtop = max(vtop, (uint32_t)*(const uint16_t*)(kb + kv_vs_off(P, D, e, tk)) & 0x7FFF);
    }
    const int ex = key_power(top);
    const uint64_t bad = __ballot(pid < 0);
    if (wave == 0) {
        float* tail = (float*)(rec + 4 * kBN * D);
        tail[lane] = pow2(ex);
        if (lane == 0) *(uint64_t*)(tail + kBN) = bad;
    }
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
        const int u = wave + 4 * e, cc = u >> 2, g = u & 3;
        const u32x4 kc = *(const u32x4*)(kb + kv_kq_unit(P, cc, g, tk));
#pragma unroll
        for (int k = 0; k < 2; ++k)
            *(u32x4*)(rec + ((8 * cc + 4 * k + g) * kBN + lane) * 16) = half_keys(kc, k, ks[2 * cc + k], pow2(-ex));
    }
    // the tokens that some row of the sequence sees: the others may hold anything
    const int lo = p.window ? len - rows - p.window + 1 : 0, tok = t0 + lane;
    const int ev = value_power(wave_top(pid >= 0 && (tok >= lo || tok < p.sinks) ? vtop : 0));
    if (tid == 0) *(int*)(rec + 4 * kBN * D + 4 * kBN + 8) = ev;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
        const int u = tid + 256 * e, m = u % 16, cc = u / 16 % (D / 32), t8 = u / (D / 2), tv = (t0 + 8 * t8) & (P - 1);
        const char* vb = head + (int64_t)max(__shfl(pid, 8 * t8, 64), 0) * kv.page_bytes;
        const u32x4 codes = *(const u32x4*)(vb + kv_vq_unit(P, D, tv >> 3, cc, m)), sc = *(const u32x4*)(vb + kv_vs_off(P, D, cc, tv));
#pragma unroll
        for (int k = 0; k < 2; ++k)
            *(u32x4*)(rec + 2 * kBN * D + (t8 * D + 32 * cc + 16 * k + m) * 16) = half_values(codes, k, sc, pow2(-ev));
    }
}

// KT = 2: two waves share 32 query rows, each with half of a tile's tokens, and
// join at the end; a workgroup then has 64 rows and a tile takes half as long.
template <int D, int KV, int W, int KT>
__global__ void __launch_bounds__(64 * W, D <= 128 ? 2 : 1) k_attn_prefill(PrefillP p) {
    constexpr int KS = D / 16, DT = D / 32, BM = 32 * W / KT, T = 64 * W;
    constexpr int NT = 2 / KT;                         // 32-token parts of a tile that a wave takes
    constexpr bool Q8 = KV == kKvQ8, STAGED = KV == kKvStaged, HALF = KV != kKvBf16;  // HALF: fp16 scores
    constexpr int NU = D / 8 / W;                      // 1 KiB units of K (and of V) that a wave copies
    constexpr int NQ8 = D / 64 * 4 / W > 0 ? D / 64 * 4 / W : 1;  // q8 units of a thread
    __shared__ __attribute__((aligned(16))) char s_k[2][kBN * D * 2], s_v[2][kBN * D * 2];
    __shared__ __attribute__((aligned(16))) float s_mul[2][kBN + 4];  // q8: what a token's scores are multiplied by
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, hf = lane >> 5;
    const KvView& kv = p.kv;
    const int seq = blockIdx.z / p.nsplit, split = blockIdx.z % p.nsplit, h = blockIdx.x, P = kv.P;
    int base, rows;
    rows_of(p, seq, base, rows);
    const int M = rows * p.G, first = (int)(gridDim.y - 1 - blockIdx.y) * BM;
    if (rows <= 0 || first >= M) return;
    const int len = min(max(p.kv_len[seq], 0), min(p.max_len, kv.max_pages << kv.plog));
    const int last = min(M, first + BM) - 1;
    const int group = wave / KT, part = wave % KT, row32 = group * 32 + c;
    const int r = min(first + row32, last), i = r / p.G;
    const int pos = len - rows + i, pfirst = len - rows + first / p.G, plast = len - rows + last / p.G;
    const size_t qat = (size_t)(base + i) * p.ldq + (size_t)(h * p.G + r % p.G) * D;

    // the query row's operand: bf16; over a q8 cache fp16 of the row divided by
    // a power of two, which comes back in `scale`
    u32x4 q[KS];
    float scale = p.scale;
    if constexpr (!HALF) {
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if (p.q_bf16) {
                q[k] = *(const u32x4*)((const uint16_t*)p.q + qat + 16 * k + 8 * hf);
            } else {
                const float* x = (const float*)p.q + qat + 16 * k + 8 * hf;
                const f32x4 a = *(const f32x4*)x, b = *(const f32x4*)(x + 4);
                q[k] = u32x4{f2bf2(a[0], a[1]), f2bf2(a[2], a[3]), f2bf2(b[0], b[1]), f2bf2(b[2], b[3])};
            }
        }
    } else {
        f32x4 x[KS][2];
        float amax = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            if (p.q_bf16) {
                const u32x4 b = *(const u32x4*)((const uint16_t*)p.q + qat + 16 * k + 8 * hf);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][e >> 2][e & 3] = as_float(e & 1 ? b[e >> 1] & 0xFFFF0000u : b[e >> 1] << 16);
            } else {
                const float* y = (const float*)p.q + qat + 16 * k + 8 * hf;
                x[k][0] = *(const f32x4*)y;
                x[k][1] = *(const f32x4*)(y + 4);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[k][e >> 2][e & 3]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 32, 64));
        const int ex = max(-100, min(100, ilogb2(amax) - 4));  // the largest value in [16, 32)
        const float down = pow2(-ex);
        scale *= pow2(ex);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            f16x8 y;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (_Float16)(x[k][e >> 2][e & 3] * down);
            q[k] = __builtin_bit_cast(u32x4, y);
        }
    }

    // the tiles any of the rows sees: the sinks' [0, ns), then [lo_t, end_t)
    const int end = plast + 1;
    const int lo = p.window ? max(0, pfirst - p.window + 1) : 0;
    const int lo_t = lo / kBN, end_t = end > 0 ? (end + kBN - 1) / kBN : 0;
    const int ns = p.window ? min(lo_t, (p.sinks + kBN - 1) / kBN) : 0;
    const int all = end > 0 ? ns + end_t - lo_t : 0;
    // this workgroup's share of them: v0 .. n - 1
    const int per = p.nsplit > 1 ? max(kPiece, (all + p.nsplit - 1) / p.nsplit) : all;
    const int v0 = min(all, split * per), n = min(all, v0 + per);
    auto tile0 = [&](int v) { return (v < ns ? v : v - ns + lo_t) * kBN; };

    // staging.  pid: the page of token tile0 + lane (-1: none)
    u32x4 rk[NQ8], rv[NQ8], rvs[NQ8];
    uint16_t rks[D / 32];
    auto page_at = [&](int v) {
        if (v >= n) return -1;
        if constexpr (STAGED) {  // the record's mask stands for the pages
            const uint64_t mask = *(const uint64_t*)(p.stage + (((size_t)seq * kv.heads + h) * p.stage_tiles + tile0(v) / kBN) * tile_record(D) + 4 * kBN * D + 4 * kBN);
            return mask >> lane & 1 ? -1 : 0;
        } else {
            return kv_page(kv, seq, tile0(v) + lane);
        }
    };
    auto fetch = [&](int v, int pid, int buf) {
        const int t0 = tile0(v) & (P - 1);  // token of the page where the tile starts (0 for pages below a tile)
        const int tk = (t0 + lane) & (P - 1);
        const char* head = kv.pages + (size_t)h * kv.head_bytes;
        if constexpr (STAGED) {
            const char* rec = p.stage + (((size_t)seq * kv.heads + h) * p.stage_tiles + tile0(v) / kBN) * tile_record(D);
#pragma unroll
            for (int e = 0; e < NU; ++e)
                copy_lds_row(rec + wave * 1024, 16 * lane + e * (W * 1024), s_k[buf] + wave * 1024 + e * (W * 1024));
#pragma unroll
            for (int e = 0; e < NU; ++e)
                copy_lds_row(rec + 2 * kBN * D + wave * 1024, 16 * lane + e * (W * 1024), s_v[buf] + wave * 1024 + e * (W * 1024));
            if (wave == 0 && lane < 17) copy_lds_row(rec + 4 * kBN * D, 16 * lane, s_mul[buf]);
        } else if constexpr (!Q8) {
            const char* kl = s_k[buf] + wave * 1024;
            const char* vl = s_v[buf] + wave * 1024;
            if (P >= kBN) {  // one page: rows of 1 KiB at addresses of the wave
                const char* pg = head + (int64_t)max(__builtin_amdgcn_readfirstlane(pid), 0) * kv.page_bytes + 16 * t0;
                const char* kb = pg + wave * (P * 16);
                const char* vb = pg + P * D * 2 + (2 * D - 16) * t0 + wave * 1024;
#pragma unroll
                for (int e = 0; e < NU; ++e)  // 8 dims of the tile's tokens
                    copy_lds_row(kb, 16 * lane + e * (W * 16) * P, kl + e * (W * 1024));
#pragma unroll
                for (int e = 0; e < NU; ++e)  // 64 dims of 8 tokens
                    copy_lds_row(vb, 16 * lane + e * (W * 1024), vl + e * (W * 1024));
            } else {
                const char* kb = head + (int64_t)max(pid, 0) * kv.page_bytes + 16 * tk + wave * (P * 16);
#pragma unroll
                for (int e = 0; e < NU; ++e) copy_lds(kb + e * (W * 16) * P, kl + e * (W * 1024));
#pragma unroll
                for (int e = 0; e < NU; ++e) {
                    const int unit = wave + W * e, t8 = unit / (D / 64), d = unit % (D / 64) * 64;
                    const char* vb = head + (int64_t)max(__builtin_amdgcn_readlane(pid, 8 * t8), 0) * kv.page_bytes;
                    copy_lds_row(vb + kv_v_unit(P, D, ((8 * t8) & (P - 1)) >> 3, d), 16 * lane, vl + e * (W * 1024));
                }
            }
        } else {
            const char* kb = head + (int64_t)max(pid, 0) * kv.page_bytes;
#pragma unroll
            for (int e = 0; e < NQ8; ++e) {
                const int u = wave + W * e;  // unit (c, g) of the lane's token
                if (u < D / 16) rk[e] = *(const u32x4*)(kb + kv_kq_unit(P, u >> 2, u & 3, tk));
            }
#pragma unroll
            for (int e = 0; e < D / 32; ++e) rks[e] = *(const uint16_t*)(kb + kv_ks_off(P, D, e, tk));
#pragma unroll
            for (int e = 0; e < NQ8; ++e) {
                const int u = tid + T * e, m = u % 16, cc = u / 16 % (D / 32), t8 = u / (D / 2);
                if (t8 < kBN / 8) {
                    const int pv = max(__shfl(pid, 8 * t8, 64), 0), tv = (t0 + 8 * t8) & (P - 1);
                    const char* vb = head + (int64_t)pv * kv.page_bytes;
                    rv[e] = *(const u32x4*)(vb + kv_vq_unit(P, D, tv >> 3, cc, m));
                    rvs[e] = *(const u32x4*)(vb + kv_vs_off(P, D, cc, tv));
                }
            }
        }
    };
    auto land = [&](int buf) {  // q8: the fetched tile, keys as fp16 over a power of two of their token, values as bf16
        if constexpr (Q8) {
            uint32_t top = 0;
#pragma unroll
            for (int e = 0; e < D / 32; ++e) top = max(top, (uint32_t)rks[e]);
            const int ex = key_power(top);
            const float down = pow2(-ex);
            if (wave == 0) s_mul[buf][lane] = pow2(ex);
#pragma unroll
            for (int e = 0; e < NQ8; ++e) {
                const int u = wave + W * e, cc = u >> 2, g = u & 3;
                if (u >= D / 16) break;
#pragma unroll
                for (int k = 0; k < 2; ++k)
                    *(u32x4*)(s_k[buf] + ((8 * cc + 4 * k + g) * kBN + lane) * 16) = half_keys(rk[e], k, rks[2 * cc + k], down);
            }
#pragma unroll
            for (int e = 0; e < NQ8; ++e) {
                const int u = tid + T * e, m = u % 16, cc = u / 16 % (D / 32), t8 = u / (D / 2);
                if (t8 >= kBN / 8) break;
#pragma unroll
                for (int k = 0; k < 2; ++k) *(u32x4*)(s_v[buf] + (t8 * D + 32 * cc + 16 * k + m) * 16) = bf16_values(rv[e], k, rvs[e]);
            }
        }
    };

    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = kNone, l = 0.f;
    // STAGED: fp16 weights are 2^15 at most, so that small ones keep their bits; o
    // is in units of the largest power of the tiles' values so far
    constexpr float kUp = STAGED ? 7.f : 0.f;
    int power = 0, power_o = -200;
    // K row of the lane in the score product (see above)
    const int krow = 16 * (c >> 4) + 8 * (c >> 2 & 1) + 4 * (c >> 3 & 1) + (c & 3);

    int pid = page_at(v0), pid_next = page_at(v0 + 1);
    if (v0 < n) {
        fetch(v0, pid, 0);
        land(0);
    }
    for (int v = v0; v < n; ++v) {
        const int buf = (v - v0) & 1, t0 = tile0(v);
        const uint64_t bad = __ballot(pid < 0);
        BQ_WAIT_VM(0);
        __syncthreads();
        pid = pid_next;
        if (v + 1 < n) fetch(v + 1, pid, buf ^ 1);
        pid_next = page_at(v + 2);
        const char* kp = s_k[buf] + (hf * kBN + 32 * NT * part + krow) * 16;
        const char* vp = s_v[buf] + ((4 * NT * part + hf) * D + c) * 16;
        // the wave that is on the matrix pipe goes first: its partner on the SIMD
        // (another workgroup's) then has the vector pipe while it waits for results
        if constexpr (!Q8) __builtin_amdgcn_s_setprio(1);
        f32x16 s[NT];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const u32x4 kf = *(const u32x4*)(kp + (2 * k * kBN + 32 * t) * 16);
                if constexpr (HALF)
                    s[t] = mfma32h(__builtin_bit_cast(f16x8, kf), __builtin_bit_cast(f16x8, q[k]), s[t]);
                else
                    s[t] = mfma32(__builtin_bit_cast(bf16x8, kf), __builtin_bit_cast(bf16x8, q[k]), s[t]);
            }
        if constexpr (!Q8) __builtin_amdgcn_s_setprio(0);
        // s[t][8u + e]: token t0 + 32 (NT part + t) + 16u + 8hf + e
        if constexpr (HALF) {
            const float* mp = s_mul[buf] + 32 * NT * part + 8 * hf;
#pragma unroll
            for (int e = 0; e < 16 * NT; e += 4) {
                const f32x4 y = *(const f32x4*)(mp + 32 * (e >> 4) + 16 * (e >> 3 & 1) + (e & 4));
#pragma unroll
                for (int x = 0; x < 4; ++x) s[e >> 4][(e & 15) + x] *= y[x];
            }
        }
        if (bad != 0 || t0 + kBN - 1 > pfirst || (p.window && t0 <= plast - p.window && t0 + kBN > p.sinks)) {
            // at an edge of what the rows see
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 32 * (NT * part + t) + 16 * (e >> 3) + 8 * hf + (e & 7), tok = t0 + at;
                    const bool me = (!(bad >> at & 1)) & (tok <= pos) & ((!p.window) | (tok > pos - p.window) | (tok < p.sinks));
                    s[t][e] = me ? s[t][e] : -INFINITY;
                }
            if (bad != 0 || t0 + kBN > end || t0 < lo) {
                // values that no row sees may hold anything: their products must not
                for (int u = tid; u < D * (kBN / 8); u += T) {
                    u32x4 mask;
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const int at = u / D * 8 + e, tok = t0 + at;
                        const bool any = (!(bad >> at & 1)) & (tok < end) & ((tok >= lo) | (tok < p.sinks));
                        const uint32_t keep = any ? (e & 1 ? 0xFFFF0000u : 0xFFFFu) : 0u;
                        mask[e >> 1] = e & 1 ? mask[e >> 1] | keep : keep;
                    }
                    *(u32x4*)(s_v[buf] + u * 16) &= mask;
                }
                __syncthreads();
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
        mx *= scale;
        if constexpr (STAGED) power = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s_mul[buf][kBN + 2]));
        if (__any(mx > m + kLazy) || (STAGED && power > power_o)) {
            const float mn = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
            float al = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
            if (STAGED && power > power_o) {
                al *= pow2(max(power_o - power, -100));
                power_o = power;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= al;
        }
        const float up = kUp - m + (STAGED ? (float)max(power - power_o, -100) : 0.f);
        float tl = 0.f;
#pragma unroll
        for (int u = 0; u < 2 * NT; ++u) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u >> 1][8 * (u & 1) + e], scale, up));
                (STAGED ? tl : l) += x[e];
            }
            const char* vf = vp + 2 * u * D * 16;
            if constexpr (STAGED) {
                f16x8 pp;
#pragma unroll
                for (int e = 0; e < 8; ++e) pp[e] = (_Float16)x[e];
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] = mfma32h(*(const f16x8*)(vf + 512 * d), pp, o[d]);
            } else {
                const bf16x8 pp = __builtin_bit_cast(bf16x8, u32x4{f2bf2(x[0], x[1]), f2bf2(x[2], x[3]), f2bf2(x[4], x[5]), f2bf2(x[6], x[7])});
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] = mfma32(*(const bf16x8*)(vf + 512 * d), pp, o[d]);
            }
        }
        if constexpr (STAGED) l = __builtin_fmaf(tl, pow2(min(power_o - power, 100)), l);
        if (v + 1 < n) land(buf ^ 1);
    }

    l += __shfl_xor(l, 32, 64);
    if (STAGED && power_o != 0 && v0 < n) {
        const float f = pow2(power_o);
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    if constexpr (KT == 2) {
        // the second part's sums to the first, through the key buffers
        float* so = (float*)s_k + group * (DT * 16 * 64) + lane;
        float* sm = (float*)s_v + group * 128 + lane;
        __syncthreads();
        if (part == 1) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) so[(16 * d + e) * 64] = o[d][e];
            sm[0] = m;
            sm[64] = l;
        }
        __syncthreads();
        if (part == 1) return;
        const float mt = fmaxf(m, sm[0]);
        const float fa = __builtin_amdgcn_exp2f(m - mt), fb = __builtin_amdgcn_exp2f(sm[0] - mt);
        l = l * fa + sm[64] * fb;
        m = mt;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] = o[d][e] * fa + so[(16 * d + e) * 64] * fb;
    }
    if (first + row32 > last) return;
    if (p.nsplit > 1) {
        const size_t to = ((size_t)split * p.n_rows + base + i) * p.q_heads + h * p.G + r % p.G;
        if (hf == 0) *(u32x2*)(p.part + p.ml + to * 2) = u32x2{__builtin_bit_cast(uint32_t, m), __builtin_bit_cast(uint32_t, l)};
        if (v0 >= n) return;  // l is 0: the row is not read
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                *(f32x4*)(p.part + to * D + 32 * d + 8 * b + 4 * hf) = f32x4{o[d][4 * b], o[d][4 * b + 1], o[d][4 * b + 2], o[d][4 * b + 3]};
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t at = (size_t)(base + i) * p.ldo + (size_t)(h * p.G + r % p.G) * D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)  // dims 32d + 8b + 4hf ..
            store4(p, at + 32 * d + 8 * b + 4 * hf, f32x4{o[d][4 * b] * inv, o[d][4 * b + 1] * inv, o[d][4 * b + 2] * inv, o[d][4 * b + 3] * inv}, l);
}

// joins the pieces of the rows, in their order: a lane has 4 dims of one row and head
template <int D>
__global__ void __launch_bounds__(256) k_attn_prefill_join(PrefillP p) {
    int base, count;
    rows_of(p, blockIdx.y, base, count);
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, in = e / (D / 4), rows = (int64_t)p.n_rows * p.q_heads;
    if (in >= (int64_t)count * p.q_heads) return;
    const int64_t at = (int64_t)base * p.q_heads + in;
    const int row = (int)(at / p.q_heads), head = (int)(at % p.q_heads), d = (int)(e % (D / 4)) * 4;
    float mt = kNone;
    for (int s = 0; s < p.nsplit; ++s) mt = fmaxf(mt, p.part[p.ml + (s * rows + at) * 2]);
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (int s = 0; s < p.nsplit; ++s) {
        const float ls = p.part[p.ml + (s * rows + at) * 2 + 1];
        if (ls == 0.f) continue;
        const float f = __builtin_amdgcn_exp2f(p.part[p.ml + (s * rows + at) * 2] - mt);
        a += *(const f32x4*)(p.part + (s * rows + at) * D + d) * f;
        l += ls * f;
    }
    store4(p, (size_t)row * p.ldo + (size_t)head * D + d, a * (l == 0.f ? 0.f : 1.f / l), l);
}

constexpr int kW = 4;  // waves of a workgroup
// 512 rows of 32 + 4 heads over 4000 tokens 84 us converting on the way, 66
// ahead; 128 rows 39 and 41, 64 rows 31 and 37
constexpr int kStageRows = 2048;

// Row tiles of 32 kW rows; of half that, shared by pairs of waves, where those
// fit the chip at once (512 rows: 19.7 us with whole tiles, 16.4 with half ones;
// 512 rows over 4000 tokens in four pieces, which do not, 59 / 78) or, where the
// tokens are not split and are several tiles, almost (the shorter rows' workgroups
// end early: 1500 rows 47 / 40, 700 rows of D 256 44 / 36; 6 x 105 rows of D 256,
// two tiles of tokens, 24 / 34)
bool half_tiles(int64_t tiles, int nsplit, int64_t steps, int slots) {
    return tiles * nsplit <= slots / 2 || (nsplit == 1 && tiles <= slots && steps >= kPiece);
}
// workgroups that the chip holds at once: two tile buffers are 64 KiB at D 128,
// 128 KiB at D 256 (counted as two there, 256 rows over 4000 tokens took 88 us
// instead of 74, 1000 rows 70 instead of 54)
int slots_of(int D, int cus) { return D <= 128 ? 2 * cus : cus; }

template <int D, int KV>
hipError_t launch_of(const PrefillP& p, int cus, hipStream_t st) {
    const int64_t rows = (int64_t)p.max_rows * p.G;
    const int64_t tiles = (rows + 32 * kW - 1) / (32 * kW), halves = (rows + 16 * kW - 1) / (16 * kW);
    hipError_t e = hipSuccess;
    if constexpr (KV == kKvStaged) {
        launch_kernel((k_stage_q8<D>), dim3(p.stage_tiles, p.kv.heads, p.kv.n_seq), dim3(256), 0, st, p);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (half_tiles(tiles * p.kv.heads * p.kv.n_seq, p.nsplit, prefill_reach(p.window, p.sinks, p.max_len) / kBN, slots_of(D, cus)))
        launch_kernel((k_attn_prefill<D, KV, kW, 2>), dim3(p.kv.heads, (uint32_t)halves, p.kv.n_seq * p.nsplit), dim3(64 * kW), 0, st, p);
    else
        launch_kernel((k_attn_prefill<D, KV, kW, 1>), dim3(p.kv.heads, (uint32_t)tiles, p.kv.n_seq * p.nsplit), dim3(64 * kW), 0, st, p);
    e = hipGetLastError();
    if (e == hipSuccess && p.nsplit > 1) {
        const int64_t n = (int64_t)p.max_rows * p.q_heads * (D / 4);
        launch_kernel((k_attn_prefill_join<D>), dim3((uint32_t)((n + 255) / 256), p.kv.n_seq), dim3(256), 0, st, p);
        e = hipGetLastError();
    }
    return e;
}
template <int D>
hipError_t launch_d(const PrefillP& p, int type, int cus, hipStream_t st) {
    if (type == kKvBf16) return launch_of<D, kKvBf16>(p, cus, st);
    return p.stage ? launch_of<D, kKvStaged>(p, cus, st) : launch_of<D, kKvQ8>(p, cus, st);
}
}  // namespace

// Pieces that the tokens of a sequence are cut into: where the row tiles leave
// workgroup slots free, as many pieces as fill them, of kPiece
// tiles at least.
int prefill_splits(int n_seq, int rows, int q_heads, int kv_heads, int D, int64_t len, int cus) {
    const int64_t tiles = ((int64_t)rows * (q_heads / kv_heads) + 32 * kW - 1) / (32 * kW) * n_seq * kv_heads;
    const int64_t steps = (len + kBN - 1) / kBN;
    return (int)std::max<int64_t>(1, std::min<int64_t>(steps / kPiece, slots_of(D, cus) / tiles));
}
// the tokens in the tiles that a window and its sinks let a row tile reach
int64_t prefill_reach(int window, int sinks, int max_len) {
    return window ? std::min<int64_t>(max_len, (int64_t)window + 32 * kW + kBN + ((int64_t)sinks + kBN - 1) / kBN * kBN) : max_len;
}
size_t prefill_part_floats(int n_rows, int q_heads, int D) { return (size_t)n_rows * q_heads * (D + 2); }

// Bytes of a q8 cache's converted tiles, 0 where they are converted as they are
// read: below kStageRows rows of a head group, or beyond 1 GiB.
size_t prefill_stage_bytes(int type, int n_seq, int rows, int q_heads, int kv_heads, int D, int max_len) {
    if (type != kKvQ8 || (int64_t)rows * (q_heads / kv_heads) < kStageRows) return 0;
    const size_t n = (size_t)n_seq * kv_heads * ((max_len + kBN - 1) / kBN) * tile_record(D);
    return n <= (size_t)1 << 30 ? n : 0;
}

hipError_t launch_attn_prefill(const KvView& kv, int type, const bq_attn_args& a, size_t stage_bytes, int nsplit, int cus, hipStream_t st) {
    PrefillP p;
    p.kv = kv;
    p.q = a.q; p.out = a.out; p.ldq = a.ldq; p.ldo = a.ldo; p.row0 = a.row0; p.kv_len = a.kv_len;
    p.stage = stage_bytes ? (char*)a.work : nullptr;
    p.stage_tiles = (a.max_len + kBN - 1) / kBN;
    p.nsplit = nsplit; p.part = (float*)((char*)a.work + stage_bytes); p.ml = (int64_t)nsplit * a.n_rows * a.q_heads * kv.D;
    p.q_heads = a.q_heads; p.G = a.q_heads / kv.heads; p.n_rows = a.n_rows; p.max_rows = std::min(a.rows, a.n_rows); p.max_len = a.max_len;
    p.window = a.window; p.sinks = a.sinks;
    p.q_bf16 = a.q_type == BQ_TYPE_BF16; p.out_bf16 = a.out_type == BQ_TYPE_BF16;
    p.scale = a.scale * 1.44269504088896341f;
    switch (kv.D) {
        case 64: return launch_d<64>(p, type, cus, st);
        case 128: return launch_d<128>(p, type, cus, st);
        default: return launch_d<256>(p, type, cus, st);
    }
}

}  // namespace bq
