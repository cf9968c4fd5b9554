// bq_attn.hip -- attention of 1..8 new tokens per sequence over the paged
// cache (decode and speculative verify), split over the cache's length.
//
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q.k_j
// in one pass over the visible tokens, with a running m.  It reads every
// visible token's K and V once per 16 query rows, so HBM bandwidth bounds it.
//
// A wave takes 32 tokens at a time and 16 query rows of one key-value head
// (the heads of the group times the new tokens).  Scores are computed
// transposed, S^T = K Q^T on 16x16x32 MFMA, so a lane holds tokens of one
// query row; the rows of the two K tiles are dealt so that lane group g holds
// tokens 8g..8g+7, which is what the second product O^T = V^T P^T takes as its
// B operand: the softmax weights never leave their lane.  The cache's layout
// is the A operands' (16 bytes per lane, 256 contiguous bytes per 16 lanes), so
// K and V go straight from HBM to registers.
//
// fp32 precision on 16-bit MFMA: K, V and int8 codes are exact in bf16, the
// codes in fp16 too.  Over a bf16 cache q and the softmax weights are sums of
// three bf16 parts (all 24 bits).  Over a q8 cache q is two fp16 parts of the
// row over a power of two (2^-22 of its largest value), a weight times a
// token's value scale two bf16 parts (2^-16 of it: a third costs 13% here,
// where the vector pipe is busy unpacking; over bf16 it costs 1%).  Every part
// has its own MFMA: the matrix pipe is far from busy.
//
// The running maximum is kept per query row and only moved when a score passes
// it by more than 2^8 (kLazy): a weight is then at most 2^8, which fp32 sums
// carry, and the accumulators are rarely rescaled.
//
// Measured (32 heads of 128 over 4): 32 sequences of 4096 to 16384 tokens in bf16
// 135 us, 4.9 TB/s of the 4.97 that a large copy reaches; one of 131072 in q8
// 38 us, 3.7 TB/s with the join's 5 us, unpacking the codes beside the reading;
// one of 777 8.4 us, two launches and a chain of loads (length, page, K and V).
#include <algorithm>

#include "bq_internal.hpp"
#include "bq_kv.hpp"

namespace bq {

namespace {
constexpr int kWaves = 4;          // per workgroup
constexpr int kRound = 512;        // 32-token steps whose pages are staged at once
constexpr float kNone = -3.402823466e38f;  // the running maximum before any token
constexpr float kLazy = 8.f;

struct DecodeP {
    KvView kv;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    const int32_t* kv_len;
    float* part;       // [n_seq][tiles][nsplit][16][D], then [..][16][2] (m, l)
    int64_t ml;        // floats before the (m, l) part
    int rows, G, tiles, nsplit, max_len, window, sinks, q_bf16, out_bf16;
    float scale;  // scale * log2(e)
};

// 32-token steps that a tile's rows at positions pfirst..plast see: the
// sinks' [0, ns), then [lo_step, lo_step + n - ns)
struct Steps {
    int lo, lo_step, ns, n;
};
BQ_DEV Steps steps_of(const DecodeP& p, int pfirst, int plast) {
    Steps s;
    s.lo = p.window ? max(0, pfirst - p.window + 1) : 0;
    s.lo_step = s.lo >> 5;
    s.ns = p.window ? min(s.lo_step, (p.sinks + 31) >> 5) : 0;
    s.n = plast < 0 ? 0 : s.ns + ((plast + 32) >> 5) - s.lo_step;
    return s;
}
BQ_DEV int length_of(const DecodeP& p, int seq) {
    return min(max(p.kv_len[seq], 0), min(p.max_len, p.kv.max_pages << p.kv.plog));
}

BQ_DEV void store4(const DecodeP& p, size_t at, f32x4 a) {
    if (p.out_bf16)
        *(u32x2*)((uint16_t*)p.out + at) = u32x2{f2bf2(a[0], a[1]), f2bf2(a[2], a[3])};
    else
        *(f32x4*)((float*)p.out + at) = a;
}
BQ_DEV f32x4 over(f32x4 a, float l) { return l == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : a * (1.f / l); }

// four int8 codes -> bf16 (exact)
BQ_DEV u32x2 codes_bf16(uint32_t w) {
    const float a = (float)(int8_t)w, b = (float)(int8_t)(w >> 8), c = (float)(int8_t)(w >> 16), d = (float)((int32_t)w >> 24);
    auto hi2 = [](float x, float y) {  // the high halves: small integers are exact in bf16
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
    };
    return u32x2{hi2(a, b), hi2(c, d)};
}
BQ_DEV bf16x8 codes8(uint32_t lo, uint32_t hi) {
    const u32x2 a = codes_bf16(lo), b = codes_bf16(hi);
    return __builtin_bit_cast(bf16x8, u32x4{a[0], a[1], b[0], b[1]});
}
BQ_DEV f16x8 codes8h(uint32_t lo, uint32_t hi) {
    f16x2 v[4];
    codes_f16(lo, v[0], v[1]);
    codes_f16(hi, v[2], v[3]);
    return f16x8{v[0][0], v[0][1], v[1][0], v[1][1], v[2][0], v[2][1], v[3][0], v[3][1]};
}
BQ_DEV f32x4 mfma16h(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
BQ_DEV f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// largest and sum over the four lane groups that share lane & 15
BQ_DEV float groups_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
BQ_DEV float groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// NQ parts of q, NP of a softmax weight
template <int D, int KV, int NQ, int NP>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) k_attn_decode(DecodeP p) {
    constexpr int KS = D / 32, DT = D / 16;
    __shared__ int s_page[kRound * 2];
    __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][D + 4];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16], s_mt[16], s_lt[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const KvView& kv = p.kv;
    const int seq = blockIdx.z, h = blockIdx.y % kv.heads, qt = blockIdx.y / kv.heads;
    const int len = length_of(p, seq);

    // the lane's query row: new token i, head r % G of the group
    const int M = p.rows * p.G, first = qt * 16, last = min(M, first + 16) - 1;
    const int pfirst = len - p.rows + first / p.G, plast = len - p.rows + last / p.G;
    const int r = min(first + c, last), i = r / p.G, pos = len - p.rows + i;
    constexpr bool Q8 = KV == kKvQ8;
    u32x4 q[NQ][KS];
    float scale = p.scale;
    {
        const size_t at = (size_t)(seq * p.rows + i) * p.ldq + (size_t)(h * p.G + r % p.G) * D + 8 * g;
        if constexpr (!Q8 && NQ == 1) {
#pragma unroll
            for (int k = 0; k < KS; ++k) q[0][k] = *(const u32x4*)((const uint16_t*)p.q + at + 32 * k);
        } else {
            float x[KS][8], amax = 0.f;
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                if (p.q_bf16) {
                    const u32x4 b = *(const u32x4*)((const uint16_t*)p.q + at + 32 * k);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[k][e] = as_float(e & 1 ? b[e >> 1] & 0xFFFF0000u : b[e >> 1] << 16);
                } else {
                    const f32x4 a = *(const f32x4*)((const float*)p.q + at + 32 * k), b = *(const f32x4*)((const float*)p.q + at + 32 * k + 4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[k][e] = a[e], x[k][4 + e] = b[e];
                }
            }
            if constexpr (Q8) {  // the row's largest value to [16, 32), but for rows of 2^-122 and less
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[k][e]));
                const int ex = max(-126, min(126, ilogb2(groups_max(amax)) - 4));
                const float down = pow2(-ex);
                scale *= pow2(ex);
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[k][e] *= down;
            }
#pragma unroll
            for (int k = 0; k < KS; ++k)
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                    if constexpr (Q8) {
                        f16x8 y;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            y[e] = (_Float16)x[k][e];
                            x[k][e] -= (float)y[e];
                        }
                        q[n][k] = __builtin_bit_cast(u32x4, y);
                    } else {
                        bf16x8 y;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            y[e] = (__bf16)x[k][e];
                            x[k][e] -= (float)y[e];
                        }
                        q[n][k] = __builtin_bit_cast(u32x4, y);
                    }
                }
        }
    }

    const Steps st = steps_of(p, pfirst, plast);
    const int end = plast + 1, lo = st.lo, n = st.n;
    const int per = (n + p.nsplit - 1) / p.nsplit;
    const int v0 = min(n, (int)blockIdx.x * per), v1 = min(n, v0 + per);

    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNone, l = 0.f;

    const bool half_pages = kv.plog == 4;  // a step spans two 16-token pages
    const int P = kv.P;
    for (int vr = v0; vr < v1; vr += kRound) {
        const int cnt = min(kRound, v1 - vr);
        __syncthreads();
        for (int e = tid; e < cnt << (half_pages ? 1 : 0); e += 256) {
            const int v = vr + (half_pages ? e >> 1 : e), ts = v < st.ns ? v : v - st.ns + st.lo_step;
            s_page[e] = kv_page(kv, seq, ts * 32 + (half_pages ? (e & 1) * 16 : 0));
        }
        __syncthreads();
        for (int w = wave; w < cnt; w += kWaves) {
            const int v = vr + w, ts = v < st.ns ? v : v - st.ns + st.lo_step, t0 = ts * 32;
            // keys: lane row c holds token 8 (c / 4) + c % 4 (+ 4 in the second tile); values: tokens 8g..
            const int gk = c >> 2;
            const int pk = half_pages ? s_page[2 * w + (gk >> 1)] : s_page[w], pv = half_pages ? s_page[2 * w + (g >> 1)] : s_page[w];
            const int ib = t0 & (P - 1);  // 0 with 16-token pages
            const int tk = ib + 8 * (half_pages ? gk & 1 : gk) + (c & 3), tv = ib + 8 * (half_pages ? g & 1 : g);
            const char* bk = kv.pages + (size_t)max(pk, 0) * kv.page_bytes + (size_t)h * kv.head_bytes;
            const char* bv = kv.pages + (size_t)max(pv, 0) * kv.page_bytes + (size_t)h * kv.head_bytes;
            // every load of the step first: the values' arrive during the scores
            u32x4 kf[2][Q8 ? KS / 2 : KS], vf[Q8 ? DT / 2 : DT], ksc[Q8 ? KS : 1], vsc[Q8 ? KS : 1];
            if constexpr (!Q8) {
#pragma unroll
                for (int k = 0; k < KS; ++k)
#pragma unroll
                    for (int t = 0; t < 2; ++t) kf[t][k] = *(const u32x4*)(bk + kv_k_unit(P, 4 * k + g, tk + 4 * t));
#pragma unroll
                for (int d = 0; d < DT; ++d) vf[d] = *(const u32x4*)(bv + kv_v_unit(P, D, tv >> 3, 16 * d + c));
            } else {
#pragma unroll
                for (int k = 0; k < KS / 2; ++k)
#pragma unroll
                    for (int t = 0; t < 2; ++t) kf[t][k] = *(const u32x4*)(bk + kv_kq_unit(P, k, g, tk + 4 * t));
#pragma unroll
                for (int k = 0; k < KS; ++k) ksc[k] = *(const u32x4*)(bv + kv_ks_off(P, D, k, tv));
#pragma unroll
                for (int d = 0; d < DT / 2; ++d) vf[d] = *(const u32x4*)(bv + kv_vq_unit(P, D, tv >> 3, d, c));
#pragma unroll
                for (int d = 0; d < DT / 2; ++d) vsc[d] = *(const u32x4*)(bv + kv_vs_off(P, D, d, tv));
            }
            __builtin_amdgcn_sched_barrier(0);
            f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    if constexpr (!Q8) {
                        const bf16x8 kb = __builtin_bit_cast(bf16x8, kf[y][k]);
#pragma unroll
                        for (int a = NQ - 1; a >= 0; --a) s[y] = mfma16(kb, __builtin_bit_cast(bf16x8, q[a][k]), s[y]);
                    } else {
                        const f16x8 kb = codes8h(kf[y][k / 2][2 * (k & 1)], kf[y][k / 2][2 * (k & 1) + 1]);
                        const uint32_t a0 = ksc[k][2 * y], a1 = ksc[k][2 * y + 1];
                        const f32x4 sc = {as_float(a0 << 16), as_float(a0 & 0xFFFF0000u), as_float(a1 << 16), as_float(a1 & 0xFFFF0000u)};
                        f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int a = NQ - 1; a >= 0; --a) x = mfma16h(kb, __builtin_bit_cast(f16x8, q[a][k]), x);
                        s[y] += x * sc;
                    }
                }
            // scores of tokens t0 + 8g + 4y + e for the lane's query rows
            const bool edge = t0 + 31 > pfirst || (p.window && t0 <= plast - p.window && t0 + 32 > p.sinks) || __any(pv < 0);
            uint32_t seen = 0xFF;  // tokens any row of the tiles sees (their values are read)
            if (edge) {
                seen = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int tok = t0 + 8 * g + e;
                    const bool any = pv >= 0 && tok < end && (tok >= lo || tok < p.sinks);
                    seen |= any ? 1u << e : 0u;
                }
                // what no row sees may hold anything: its products must not
                if constexpr (!Q8) {
                    u32x4 mask;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        mask[e] = (seen >> (2 * e) & 1 ? 0xFFFFu : 0u) | (seen >> (2 * e + 1) & 1 ? 0xFFFF0000u : 0u);
#pragma unroll
                    for (int d = 0; d < DT; ++d) vf[d] &= mask;
                }
            }
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = s[e >> 2][e & 3] * scale;
            if (edge) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int tok = t0 + 8 * g + e;
                    const bool me = pv >= 0 && tok <= pos && (!p.window || tok > pos - p.window || tok < p.sinks);
                    x[e] = me ? x[e] : -INFINITY;
                }
            }
            float mx = x[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) mx = fmaxf(mx, x[e]);
            if (__any(mx > m + kLazy)) {
                const float mn = fmaxf(m, groups_max(mx));
                const float al = __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= al;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= al;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = __builtin_amdgcn_exp2f(x[e] - m);
                l += x[e];
            }
            auto parts = [&](const float (&y)[8], bf16x8 (&pp)[NP]) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float z = y[e];
#pragma unroll
                    for (int a = 0; a < NP; ++a) {
                        const __bf16 w = (__bf16)z;
                        pp[a][e] = w;
                        z -= (float)w;
                    }
                }
            };
            bf16x8 pp[NP];
            if constexpr (!Q8) {
                parts(x, pp);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int a = NP - 1; a >= 0; --a) o[d] = mfma16(__builtin_bit_cast(bf16x8, vf[d]), pp[a], o[d]);
            } else {
#pragma unroll
                for (int d = 0; d < DT / 2; ++d) {
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float vs = as_float(e & 1 ? vsc[d][e >> 1] & 0xFFFF0000u : vsc[d][e >> 1] << 16);
                        y[e] = x[e] * (edge && !(seen >> e & 1) ? 0.f : vs);  // codes are finite, an unseen scale may not be
                    }
                    parts(y, pp);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int a = NP - 1; a >= 0; --a)
                            o[2 * d + u] = mfma16(codes8(vf[d][2 * u], vf[d][2 * u + 1]), pp[a], o[2 * d + u]);
                }
            }
        }
    }

    // join the waves
    l = groups_sum(l);
    if (g == 0) {
        s_m[wave][c] = m;
        s_l[wave][c] = l;
    }
    __syncthreads();
    float mt = s_m[0][c], lt = 0.f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) mt = fmaxf(mt, s_m[w][c]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) lt += s_l[w][c] * __builtin_amdgcn_exp2f(s_m[w][c] - mt);
    const float f = __builtin_amdgcn_exp2f(m - mt);
#pragma unroll
    for (int d = 0; d < DT; ++d) *(f32x4*)&s_o[wave][c][16 * d + 4 * g] = o[d] * f;
    if (wave == 0 && g == 0) {
        s_mt[c] = mt;
        s_lt[c] = lt;
    }
    __syncthreads();
    const size_t piece = ((size_t)seq * p.tiles + blockIdx.y) * p.nsplit + blockIdx.x;
    for (int e = tid; e < 16 * (D / 4); e += 256) {
        const int row = e / (D / 4), d = e % (D / 4) * 4, r = first + row;
        if (r > last) continue;
        f32x4 a = *(const f32x4*)&s_o[0][row][d];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) a += *(const f32x4*)&s_o[w][row][d];
        if (p.nsplit > 1) {
            const size_t at = piece * 16 + row;
            *(f32x4*)(p.part + at * D + d) = a;
            if (d == 0) {
                p.part[p.ml + at * 2] = s_mt[row];
                p.part[p.ml + at * 2 + 1] = s_lt[row];
            }
        } else {
            store4(p, (size_t)(seq * p.rows + r / p.G) * p.ldo + (size_t)(h * p.G + r % p.G) * D + d, over(a, s_lt[row]));
        }
    }
}

// joins the pieces of one query row: D / 4 lanes per piece, the pieces dealt
// over the rest of the workgroup's T lanes, in a fixed order
template <int D, int T>
__global__ void __launch_bounds__(T) k_attn_join(DecodeP p) {
    constexpr int L = D / 4, S = T / L;
    __shared__ __attribute__((aligned(16))) float s_o[S][D];
    __shared__ float s_l[S], s_mx[T / 64];
    const int ht = p.kv.heads, tid = threadIdx.x;
    const int row = blockIdx.x, h = blockIdx.y, seq = blockIdx.z;
    const size_t tile = (size_t)seq * p.tiles + (size_t)(row / 16) * ht + h, at0 = tile * p.nsplit * 16 + row % 16;
    const float* ml = p.part + p.ml + at0 * 2;
    float mt = kNone;
    for (int s = tid; s < p.nsplit; s += T) mt = fmaxf(mt, ml[s * 32]);
    for (int d = 1; d < 64; d <<= 1) mt = fmaxf(mt, __shfl_xor(mt, d, 64));
    if ((tid & 63) == 0) s_mx[tid >> 6] = mt;
    __syncthreads();
    for (int w = 0; w < T / 64; ++w) mt = fmaxf(mt, s_mx[w]);
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    float lt = 0.f;
#pragma unroll 4
    for (int s = tid / L; s < p.nsplit; s += S) {
        const float l = ml[s * 32 + 1];
        const float f = __builtin_amdgcn_exp2f(ml[s * 32] - mt);
        a += *(const f32x4*)(p.part + (at0 + (size_t)s * 16) * D + tid % L * 4) * f;
        lt += l * f;
    }
    *(f32x4*)&s_o[tid / L][tid % L * 4] = a;
    if (tid % L == 0) s_l[tid / L] = lt;
    __syncthreads();
    if (tid >= L) return;
    for (int s = 1; s < S; ++s) {
        a += *(const f32x4*)&s_o[s][tid * 4];
        lt += s_l[s];
    }
    store4(p, (size_t)(seq * p.rows + row / p.G) * p.ldo + (size_t)(h * p.G + row % p.G) * D + tid * 4, over(a, lt));
}

template <int D, int KV>
hipError_t launch_decode_of(const DecodeP& p, hipStream_t st) {
    const dim3 grid(p.nsplit, p.tiles, p.kv.n_seq);
    if (p.q_bf16 && p.out_bf16)
        launch_kernel((k_attn_decode<D, KV, 1, 1>), grid, dim3(256), 0, st, p);
    else
        launch_kernel((k_attn_decode<D, KV, KV == kKvQ8 ? 2 : 3, KV == kKvQ8 ? 2 : 3>), grid, dim3(256), 0, st, p);
    if (p.nsplit > 1) {
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        // more than 32 pieces keep 1024 lanes busy; fewer leave them idle
        const dim3 rows(p.rows * p.G, p.kv.heads, p.kv.n_seq);
        if (p.nsplit > 32)
            launch_kernel((k_attn_join<D, 1024>), rows, dim3(1024), 0, st, p);
        else
            launch_kernel((k_attn_join<D, 256>), rows, dim3(256), 0, st, p);
    }
    return hipGetLastError();
}
// 16-row tiles of a key-value head's query rows, each a workgroup of its own:
// a wave with two tiles on the same tokens reads them once, but half as many
// waves read (8 sequences x 8 rows of 8 heads over 9001 tokens: 49 us with two,
// 43 us with one)
int q_tiles(int rows, int G) { return (rows * G + 15) / 16; }
}  // namespace

// Pieces that the `len` tokens of a sequence that its rows see are cut into: two
// workgroups per CU, each wave at least one 32-token step.  (At D 256 one fits a CU
// in all forms but a bf16 cache's with bf16 in and out, so the pieces of a long
// sequence run in two rounds there.)  A few steps are not
// cut, as the join is a launch of its own (2.5 us) and a step costs what its
// bytes do, a q8 one twice that: 512 tokens of bf16 D 128 take 7.8 us whole and
// 8.3 in four pieces, 777 10.9 and 8.4; D 64 5.7 / 7.5 and 8.1 / 8.1; D 256 11.5
// / 10.6; q8 D 128, 256 tokens 7.5 / 8.9, 512 10.8 / 9.1
int decode_splits(int type, int n_seq, int rows, int q_heads, int kv_heads, int D, int64_t len, int cus) {
    const int64_t tiles = (int64_t)n_seq * kv_heads * q_tiles(rows, q_heads / kv_heads);
    const int64_t each = ((len + 31) / 32 + kWaves - 1) / kWaves;  // steps of a wave
    if (each * D * (type == kKvQ8 ? 2 : 1) <= 512) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(each, 2 * cus / tiles));
}
// the tokens in the steps that a window and its sinks reach
int64_t decode_reach(int rows, int window, int sinks, int max_len) {
    return window ? std::min<int64_t>(max_len, (int64_t)window + rows + 30 + ((int64_t)sinks + 31) / 32 * 32) : max_len;
}

size_t decode_part_floats(int n_seq, int rows, int q_heads, int kv_heads, int D) {
    return (size_t)n_seq * kv_heads * q_tiles(rows, q_heads / kv_heads) * 16 * (D + 2);
}

hipError_t launch_attn_decode(const KvView& kv, int type, const bq_attn_args& a, int nsplit, hipStream_t st) {
    DecodeP p;
    p.kv = kv;
    p.q = a.q; p.out = a.out; p.ldq = a.ldq; p.ldo = a.ldo; p.kv_len = a.kv_len;
    p.rows = a.rows; p.G = a.q_heads / kv.heads; p.tiles = kv.heads * q_tiles(p.rows, p.G);
    p.nsplit = nsplit; p.max_len = a.max_len; p.window = a.window; p.sinks = a.sinks;
    p.q_bf16 = a.q_type == BQ_TYPE_BF16; p.out_bf16 = a.out_type == BQ_TYPE_BF16;
    p.scale = a.scale * 1.44269504088896341f;
    p.part = (float*)a.work;
    p.ml = (int64_t)kv.n_seq * p.tiles * nsplit * 16 * kv.D;
    const bool q8 = type == kKvQ8;
    switch (kv.D) {
        case 64: return q8 ? launch_decode_of<64, kKvQ8>(p, st) : launch_decode_of<64, kKvBf16>(p, st);
        case 128: return q8 ? launch_decode_of<128, kKvQ8>(p, st) : launch_decode_of<128, kKvBf16>(p, st);
        default: return q8 ? launch_decode_of<256, kKvQ8>(p, st) : launch_decode_of<256, kKvBf16>(p, st);
    }
}

}  // namespace bq
