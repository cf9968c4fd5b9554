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
// bf16; q8 is dequantized to bf16 on the way) while the one before is computed.
#include <algorithm>

#include "bq_internal.hpp"
#include "bq_kv.hpp"

namespace bq {

namespace {
constexpr int kBM = 128;         // query rows of a workgroup
constexpr int kBN = 64;          // tokens of a tile
constexpr float kNone = -1e30f;  // the running maximum before any token
constexpr float kLazy = 8.f;     // it moves when a score passes it by more (log2)

struct PrefillP {
    KvView kv;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    const int32_t* row0;
    const int32_t* kv_len;
    int G, n_rows, max_rows, max_len, window, sinks, q_bf16, out_bf16;
    float scale;  // scale * log2(e)
};

BQ_DEV f32x16 mfma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// 16 bytes per lane straight to LDS at lds + 16 * lane (m0: see bq_gemm.hip's dma16)
BQ_DEV void copy_lds(const void* src, const void* lds) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds);
    asm volatile("s_mov_b32 m0, %1\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(src), "s"(m0) : "m0", "memory");
}

BQ_DEV u32x2 dequant4(uint32_t w, float a, float b, float c, float d) {
    return u32x2{f2bf2((float)(int8_t)w * a, (float)(int8_t)(w >> 8) * b),
                 f2bf2((float)(int8_t)(w >> 16) * c, (float)((int32_t)w >> 24) * d)};
}

template <int D, int KV>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) k_attn_prefill(PrefillP p) {
    constexpr int KS = D / 16, DT = D / 32;
    __shared__ __attribute__((aligned(16))) char s_k[2][kBN * D * 2], s_v[2][kBN * D * 2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 31, hf = lane >> 5;
    const KvView& kv = p.kv;
    const int seq = blockIdx.z, h = blockIdx.y, P = kv.P;
    const int b0 = p.row0 ? p.row0[seq] : 0, b1 = p.row0 ? p.row0[seq + 1] : p.n_rows;
    // a sequence's rows, kept inside the buffers whatever row0 holds
    const int base = min(max(b0, 0), p.n_rows), rows = min(min(max(b1, 0), p.n_rows) - base, p.max_rows);
    const int M = rows * p.G, first = (int)(gridDim.x - 1 - blockIdx.x) * kBM;
    if (rows <= 0 || first >= M) return;
    const int len = min(max(p.kv_len[seq], 0), min(p.max_len, kv.max_pages << kv.plog));
    const int last = min(M, first + kBM) - 1;
    const int r = min(first + wave * 32 + c, last), i = r / p.G;
    const int pos = len - rows + i, pfirst = len - rows + first / p.G, plast = len - rows + last / p.G;
    const size_t qat = (size_t)(base + i) * p.ldq + (size_t)(h * p.G + r % p.G) * D;

    bf16x8 q[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
        if (p.q_bf16) {
            q[k] = *(const bf16x8*)((const uint16_t*)p.q + qat + 16 * k + 8 * hf);
        } else {
            const float* x = (const float*)p.q + qat + 16 * k + 8 * hf;
            const f32x4 a = *(const f32x4*)x, b = *(const f32x4*)(x + 4);
            q[k] = __builtin_bit_cast(bf16x8, u32x4{f2bf2(a[0], a[1]), f2bf2(a[2], a[3]), f2bf2(b[0], b[1]), f2bf2(b[2], b[3])});
        }
    }

    // the tiles any of the rows sees: the sinks' [0, ns), then [lo_t, end_t)
    const int end = plast + 1;
    const int lo = p.window ? max(0, pfirst - p.window + 1) : 0;
    const int lo_t = lo / kBN, end_t = end > 0 ? (end + kBN - 1) / kBN : 0;
    const int ns = p.window ? min(lo_t, (p.sinks + kBN - 1) / kBN) : 0;
    const int n = end > 0 ? ns + end_t - lo_t : 0;
    auto tile0 = [&](int v) { return (v < ns ? v : v - ns + lo_t) * kBN; };

    // staging.  pid: the page of token tile0 + lane (-1: none)
    u32x4 rk[D / 64], rv[D / 64], rvs[D / 64];
    uint16_t rks[D / 32];
    auto page_at = [&](int v) { return v < n ? kv_page(kv, seq, tile0(v) + lane) : -1; };
    auto fetch = [&](int v, int pid, int buf) {
        const int t0 = tile0(v) & (P - 1);  // token of the page where the tile starts (0 for pages below a tile)
        const int tk = (t0 + lane) & (P - 1);
        const char* kb = kv.pages + (size_t)max(pid, 0) * kv.page_bytes + (size_t)h * kv.head_bytes;
        if constexpr (KV == kKvBf16) {
#pragma unroll
            for (int e = 0; e < D / 32; ++e) {  // 8 dims of the tile's tokens
                const int ch = wave + 4 * e;
                copy_lds(kb + kv_k_unit(P, ch, tk), s_k[buf] + ch * 1024);
            }
#pragma unroll
            for (int e = 0; e < D / 32; ++e) {  // 64 dims of 8 tokens
                const int unit = wave + 4 * e, t8 = unit / (D / 64), d = unit % (D / 64) * 64 + lane;
                const int pv = max(__shfl(pid, 8 * t8, 64), 0);
                const char* vb = kv.pages + (size_t)pv * kv.page_bytes + (size_t)h * kv.head_bytes;
                copy_lds(vb + kv_v_unit(P, D, ((t0 + 8 * t8) & (P - 1)) >> 3, d), s_v[buf] + unit * 1024);
            }
        } else {
#pragma unroll
            for (int e = 0; e < D / 64; ++e) rk[e] = *(const u32x4*)(kb + kv_kq_unit(P, e, wave, tk));
#pragma unroll
            for (int e = 0; e < D / 32; ++e) rks[e] = *(const uint16_t*)(kb + kv_ks_off(P, D, e, tk));
#pragma unroll
            for (int e = 0; e < D / 64; ++e) {
                const int u = tid + 256 * e, m = u % 16, cc = u / 16 % (D / 32), t8 = u / (D / 2);
                const int pv = max(__shfl(pid, 8 * t8, 64), 0), tv = (t0 + 8 * t8) & (P - 1);
                const char* vb = kv.pages + (size_t)pv * kv.page_bytes + (size_t)h * kv.head_bytes;
                rv[e] = *(const u32x4*)(vb + kv_vq_unit(P, D, tv >> 3, cc, m));
                rvs[e] = *(const u32x4*)(vb + kv_vs_off(P, D, cc, tv));
            }
        }
    };
    auto land = [&](int buf) {  // q8: the fetched tile as bf16
        if constexpr (KV == kKvQ8) {
#pragma unroll
            for (int e = 0; e < D / 64; ++e)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float s = bf2f(rks[2 * e + k]);
                    const u32x2 a = dequant4(rk[e][2 * k], s, s, s, s), b = dequant4(rk[e][2 * k + 1], s, s, s, s);
                    *(u32x4*)(s_k[buf] + ((8 * e + 4 * k + wave) * kBN + lane) * 16) = u32x4{a[0], a[1], b[0], b[1]};
                }
#pragma unroll
            for (int e = 0; e < D / 64; ++e) {
                const int u = tid + 256 * e, m = u % 16, cc = u / 16 % (D / 32), t8 = u / (D / 2);
                float s[8];
#pragma unroll
                for (int x = 0; x < 8; ++x) s[x] = as_float(x & 1 ? rvs[e][x >> 1] & 0xFFFF0000u : rvs[e][x >> 1] << 16);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const u32x2 a = dequant4(rv[e][2 * k], s[0], s[1], s[2], s[3]), b = dequant4(rv[e][2 * k + 1], s[4], s[5], s[6], s[7]);
                    *(u32x4*)(s_v[buf] + (t8 * D + 32 * cc + 16 * k + m) * 16) = u32x4{a[0], a[1], b[0], b[1]};
                }
            }
        }
    };

    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
    float m = kNone, l = 0.f;
    // K row of the lane in the score product (see above)
    const int krow = 16 * (c >> 4) + 8 * (c >> 2 & 1) + 4 * (c >> 3 & 1) + (c & 3);

    int pid = page_at(0), pid_next = page_at(1);
    if (n > 0) fetch(0, pid, 0);
    if (n > 0) land(0);
    for (int v = 0; v < n; ++v) {
        const int buf = v & 1, t0 = tile0(v);
        const uint64_t bad = __ballot(pid < 0);
        BQ_WAIT_VM(0);
        __syncthreads();
        pid = pid_next;
        if (v + 1 < n) fetch(v + 1, pid, buf ^ 1);
        pid_next = page_at(v + 2);

        f32x16 s[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int e = 0; e < 16; ++e) s[t][e] = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k)
                s[t] = mfma32(*(const bf16x8*)(s_k[buf] + ((2 * k + hf) * kBN + 32 * t + krow) * 16), q[k], s[t]);
        }
        const bool edge = bad != 0 || t0 + kBN - 1 > pfirst || (p.window && t0 <= plast - p.window && t0 + kBN > p.sinks);
        // s[t][8u + e]: token t0 + 32t + 16u + 8hf + e
        if (edge) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 32 * t + 16 * (e >> 3) + 8 * hf + (e & 7), tok = t0 + at;
                    const bool me = !(bad >> at & 1) && tok <= pos && (!p.window || tok > pos - p.window || tok < p.sinks);
                    s[t][e] = me ? s[t][e] : -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = fmaxf(mx, s[t][e]);
        mx *= p.scale;
        if (__any(mx > m + kLazy)) {
            const float mn = fmaxf(m, fmaxf(mx, __shfl_xor(mx, 32, 64)));
            const float al = __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= al;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= al;
        }
        bf16x8 pp[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * u + e], p.scale, -m));
                    l += x[e];
                }
                pp[2 * t + u] = __builtin_bit_cast(bf16x8, u32x4{f2bf2(x[0], x[1]), f2bf2(x[2], x[3]), f2bf2(x[4], x[5]), f2bf2(x[6], x[7])});
            }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            u32x4 mask = {~0u, ~0u, ~0u, ~0u};
            if (edge) {
                // what no row sees may hold anything: its products must not
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int at = 16 * u + 8 * hf + e, tok = t0 + at;
                    const bool any = !(bad >> at & 1) && tok < end && (tok >= lo || tok < p.sinks);
                    if (!any) mask[e >> 1] &= e & 1 ? 0xFFFFu : 0xFFFF0000u;
                }
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                u32x4 vf = *(const u32x4*)(s_v[buf] + ((2 * u + hf) * D + 32 * d + c) * 16);
                if (edge) vf &= mask;
                o[d] = mfma32(__builtin_bit_cast(bf16x8, vf), pp[u], o[d]);
            }
        }
        if (v + 1 < n) land(buf ^ 1);
    }

    l += __shfl_xor(l, 32, 64);
    if (first + wave * 32 + c > last) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const size_t at = (size_t)(base + i) * p.ldo + (size_t)(h * p.G + r % p.G) * D;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b) {  // dims 32d + 8b + 4hf ..
            f32x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = l == 0.f ? 0.f : o[d][4 * b + e] * inv;
            const size_t to = at + 32 * d + 8 * b + 4 * hf;
            if (p.out_bf16)
                *(u32x2*)((uint16_t*)p.out + to) = u32x2{f2bf2(y[0], y[1]), f2bf2(y[2], y[3])};
            else
                *(f32x4*)((float*)p.out + to) = y;
        }
}

template <int D, int KV>
hipError_t launch_of(const PrefillP& p, hipStream_t st) {
    const int64_t tiles = ((int64_t)p.max_rows * p.G + kBM - 1) / kBM;
    launch_kernel((k_attn_prefill<D, KV>), dim3((uint32_t)tiles, p.kv.heads, p.kv.n_seq), dim3(256), 0, st, p);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_attn_prefill(const KvView& kv, int type, const bq_attn_args& a, hipStream_t st) {
    PrefillP p;
    p.kv = kv;
    p.q = a.q; p.out = a.out; p.ldq = a.ldq; p.ldo = a.ldo; p.row0 = a.row0; p.kv_len = a.kv_len;
    p.G = a.q_heads / kv.heads; p.n_rows = a.n_rows; p.max_rows = std::min(a.rows, a.n_rows); p.max_len = a.max_len;
    p.window = a.window; p.sinks = a.sinks;
    p.q_bf16 = a.q_type == BQ_TYPE_BF16; p.out_bf16 = a.out_type == BQ_TYPE_BF16;
    p.scale = a.scale * 1.44269504088896341f;
    const bool q8 = type == kKvQ8;
    switch (kv.D) {
        case 64: return q8 ? launch_of<64, kKvQ8>(p, st) : launch_of<64, kKvBf16>(p, st);
        case 128: return q8 ? launch_of<128, kKvQ8>(p, st) : launch_of<128, kKvBf16>(p, st);
        default: return q8 ? launch_of<256, kKvQ8>(p, st) : launch_of<256, kKvBf16>(p, st);
    }
}

}  // namespace bq
