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
// of two first, so that rows of any size keep 2^-11 of their largest value.  Where
// the q8 tiles are converted ahead of the attention (k_stage_q8), values and weights
// are fp16 too, 2^-11 of each instead of 2^-8, for 4% of the time, as long as every
// scale of a tile lies in a window that fp16 holds (plain_scale).  A workgroup that
// meets another tile starts again (kKvCodes), with the values as codes and their
// scales in the weights.
//
// Few rows over many tokens are split over workgroups (prefill_splits) and joined
// in the pieces' order; a short chunk halves the row tiles (half_tiles).
// Measured (32 heads of 128 over 4, bf16): 8192 rows 557 us, 986 TFLOP/s of the
// 1187 that a large library product reaches; 512 rows 15.7 us, eight dependent tiles
// on half of the workgroup slots, the launch, the first tile's latency (page, then K
// and V) and the epilogue.
// Five ragged chunks of up to 700 rows over a q8 cache, window 2048: 180 us for
// 77.7 GFLOP; the 584 row tiles fill 512 slots once and then 72 of them again (and
// are not split, as prefill_splits counts n_seq times the longest chunk: 880).
#include <algorithm>

#include "bq_internal.hpp"
#include "bq_kv.hpp"

namespace bq {

namespace {
constexpr int kBN = 64;          // tokens of a tile
// a q8 cache's tiles turned into the products' operands ahead of the attention:
// fp16 keys and values as they lie in LDS, what the tokens' scores are
// multiplied by, the mask of unmapped tokens, whether fp16 holds the values
constexpr int kKvStaged = 2;
// q8 tiles converted on the way, values as codes: for rows that fp16 values do not serve
constexpr int kKvCodes = 3;
constexpr int64_t tile_record(int D) { return 4 * kBN * D + 512; }
constexpr int kPiece = 8;        // tiles of a piece at least, where the tokens are split
constexpr float kNone = -3.402823466e38f;  // the running maximum before any token
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
BQ_DEV int key_power(uint32_t top) { return max(-126, min(126, (int)(top >> 7) - 127)); }
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
// Whether fp16 serves a q8 value of this scale (bf16 bits): 0, or 2^-18 <= scale < 2.
// Values are stored times 2^kLift: a code times its scale is then 2^-10 to 2^16 and
// keeps 2^-11 of itself.  Weights are fp16 beside them, 2^10 at the row's largest
// (kUp), and one below 2^-24 of that is off by 2^-35 of it: with 2^19 between the
// scales and 2^7 of a code this stays below 2^-9 of the largest weight's own scale.
// A wider window, or one that moves from tile to tile, would lose that: a value that
// a row gives no weight must not cost the others bits.
// A workgroup that meets a tile with any other scale starts again with the values as
// codes, in bf16 (exact), and each weight times the token's scale, as two bf16 parts,
// for each 32 dims (kKvCodes): 2^-16 of each term at any size.  Starting again keeps
// the loops, and their registers, apart: with both forms of a tile in one loop 39
// registers spill, and five chunks of up to 700 rows take 206 us instead of 184; a
// second launch for the rows left takes 194 with none left.  8192 rows take 620 us, and
// 1585 where every tile is of that kind.
constexpr int kLift = 8;
BQ_DEV bool plain_scale(uint32_t bits) {
    const uint32_t a = bits & 0x7FFF;
    return a == 0 || (a >= 0x3680 && a < 0x4000);
}
// 8 tokens' codes of a value's dim times their scales and 2^kLift
BQ_DEV u32x4 half_values(u32x4 codes, int k, u32x4 scales) {
    constexpr float up = 1 << kLift;
    f16x2 lo, hi;
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        codes_f16(codes[2 * k + w], lo, hi);
        const uint32_t a = scales[2 * w], b = scales[2 * w + 1];
        r[2 * w] = __builtin_bit_cast(uint32_t, lo * f16x2{(_Float16)(as_float(a << 16) * up), (_Float16)(as_float(a & 0xFFFF0000u) * up)});
        r[2 * w + 1] = __builtin_bit_cast(uint32_t, hi * f16x2{(_Float16)(as_float(b << 16) * up), (_Float16)(as_float(b & 0xFFFF0000u) * up)});
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
    // the tokens that some row of the sequence sees: the others may hold anything
    const int lo = p.window ? len - rows - p.window + 1 : 0, tok = t0 + lane;
    const bool seen = pid >= 0 && (tok >= lo || tok < p.sinks);
    uint16_t ks[D / 32];
    uint32_t top = 0;  // the token's largest key scale
    bool plain = true;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) {
        ks[e] = *(const uint16_t*)(kb + kv_ks_off(P, D, e, tk));
        top = max(top, (uint32_t)ks[e]);
        plain = plain && plain_scale(*(const uint16_t*)(kb + kv_vs_off(P, D, e, tk)));
    }
    const int ex = key_power(top);
    const bool odd = __any(seen && !plain);  // the same in every wave
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
    if (tid == 0) *(int*)(rec + 4 * kBN * D + 4 * kBN + 8) = odd;
#pragma unroll
    for (int e = 0; e < D / 64; ++e) {
        const int u = tid + 256 * e, m = u % 16, cc = u / 16 % (D / 32), t8 = u / (D / 2), tv = (t0 + 8 * t8) & (P - 1);
        const char* vb = head + (int64_t)max(__shfl(pid, 8 * t8, 64), 0) * kv.page_bytes;
        const u32x4 codes = *(const u32x4*)(vb + kv_vq_unit(P, D, tv >> 3, cc, m)), sc = *(const u32x4*)(vb + kv_vs_off(P, D, cc, tv));
#pragma unroll
        for (int k = 0; k < 2; ++k)
            *(u32x4*)(rec + 2 * kBN * D + (t8 * D + 32 * cc + 16 * k + m) * 16) = half_values(codes, k, sc);
    }
}

// KT = 2: two waves share 32 query rows, each with half of a tile's tokens, and
// join at the end; a workgroup then has 64 rows and a tile takes half as long.
template <int D, int W, int KT>
BQ_DEV void attend_codes(const PrefillP& p, char (&s_k)[2][kBN * D * 2], char (&s_v)[2][kBN * D * 2], float (&s_mul)[2][kBN + 4],
                         uint16_t (&s_vs)[2][D / 32 * kBN]) {
    constexpr int KV = kKvCodes;
#include "bq_attn_prefill_rows.inc"
}

template <int D, int KV, int W, int KT>
__global__ void __launch_bounds__(64 * W, D <= 128 ? 2 : 1) k_attn_prefill(PrefillP p) {
    __shared__ __attribute__((aligned(16))) char s_k[2][kBN * D * 2], s_v[2][kBN * D * 2];
    __shared__ __attribute__((aligned(16))) float s_mul[2][kBN + 4];         // q8: what a token's scores are multiplied by
    __shared__ __attribute__((aligned(16))) uint16_t s_vs[2][D / 32 * kBN];  // kKvCodes: the values' scales
#include "bq_attn_prefill_rows.inc"
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
    const size_t n = (size_t)n_seq * kv_heads * (((int64_t)max_len + kBN - 1) / kBN) * tile_record(D);
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
