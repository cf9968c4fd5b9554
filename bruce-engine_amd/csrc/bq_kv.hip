// bq_kv.hip -- a step's QKV rows into the paged cache (per-head RMS norm,
// rotation, bf16 or q8 storage), the rotated queries, and the cache read back.
//
// n(x) = x * rsqrt(sum x^2 / D + eps) * w, then (a, b) -> (a c - b s, b c + a s)
// on the rotated pairs.  Everything is one pass over the rows: fp32 in, the
// queries and the cache's bytes out, so the floor is their bytes.
//
// A lane holds the 8 values of four rotation pairs (two 16-byte loads), so a
// head is D/8 neighbouring lanes: the rotation stays inside a lane and the
// norm's sum is a butterfly over them.  Keys and values go through LDS as fp32
// rows, because the cache stores 8 tokens of one dim together (values) and a
// 32-value group's scale needs the whole group: a workgroup takes 16 rows of
// one head, and rows that are 8 neighbouring tokens of a page (a prompt) leave
// as whole 16-byte units; others as single elements.
//
// Bounds: a prompt its bytes (8192 rows of 32 + 4 + 4 heads of 128: 250 MB,
// 50 us, 5 TB/s, what a large copy reaches; 58 us where the outputs and inputs of
// other calls have passed through the cache); one token the launch and the chain
// position -> page -> store (3.7 us).
#include "bq_internal.hpp"
#include "bq_kv.hpp"

namespace bq {

namespace {
constexpr int kFewRows = 1024;

struct AppendP {
    KvView kv;
    const float* x[3];  // q, k, v
    int64_t ld[3];
    const float* w[2];  // q, k norm weights or NULL
    const int32_t* pos;
    const int32_t* seq;
    const float* rope;
    void* q_out;
    float eps;
    int rows, q_heads, rot, n_pos, interleaved, q_bf16, kv_blocks;
};

// offsets of a lane's two quads in the head and whether they are rotated; the
// rotation's cosines are rope[4j..4j+3] in either order of the pairs
BQ_DEV bool quad_offsets(const AppendP& p, int j, int& oa, int& ob) {
    if (p.interleaved) {
        oa = 8 * j;
        ob = oa + 4;
        return 8 * j < p.rot;
    }
    if (8 * j < p.rot) {
        oa = 4 * j;
        ob = oa + p.rot / 2;
        return true;
    }
    oa = 8 * j;  // past the rotated part: 8 values in order
    ob = oa + 4;
    return false;
}

// the lane's quads of one head, normed (w != NULL) and rotated (turn)
template <int D>
BQ_DEV void norm_turn(const AppendP& p, const float* w, bool turn, int pos, int oa, int ob, int j, f32x4& a, f32x4& b) {
    f32x4 c, s;
    if (turn) {
        const float* cs = p.rope + (size_t)pos * p.rot + 4 * j;
        c = *(const f32x4*)cs;
        s = *(const f32x4*)(cs + p.rot / 2);
    }
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) ss += a[e] * a[e] + b[e] * b[e];
#pragma unroll
        for (int d = 1; d < D / 8; d <<= 1) ss += __shfl_xor(ss, d, 64);
        const float k = 1.0f / sqrtf(ss * (1.0f / D) + p.eps);
        const f32x4 wa = *(const f32x4*)(w + oa), wb = *(const f32x4*)(w + ob);
        a = a * k * wa;
        b = b * k * wb;
    }
    if (turn) {
        if (p.interleaved) {
            const f32x4 x = a, y = b;
            a = f32x4{x[0] * c[0] - x[1] * s[0], x[1] * c[0] + x[0] * s[0], x[2] * c[1] - x[3] * s[1], x[3] * c[1] + x[2] * s[1]};
            b = f32x4{y[0] * c[2] - y[1] * s[2], y[1] * c[2] + y[0] * s[2], y[2] * c[3] - y[3] * s[3], y[3] * c[3] + y[2] * s[3]};
        } else {
            const f32x4 x = a;
            a = x * c - b * s;
            b = b * c + x * s;
        }
    }
}

// 1 / d of a bf16 scale (0 for an all-zero group, and for one that holds a NaN or an
// infinity, which stay in the scale).  Below 2^-120 it may pass fp32's range: then
// minus 1 / (2^24 d), against which the values are taken times -2^24.
BQ_DEV float scale_of(float amax, uint16_t& bits) {
    bits = f2bf(amax * (1.f / 127.f));
    const float d = bf2f(bits);
    return d >= 0x1p-120f ? 1.f / d : d > 0.f ? -1.f / (d * 0x1p24f) : 0.f;
}
BQ_DEV uint32_t code_of(float x, float inv) {
    const float y = inv < 0.f ? x * -0x1p24f : x;
    return (uint32_t)(int)rintf(__builtin_amdgcn_fmed3f(y * inv, -127.f, 127.f)) & 0xFF;
}

template <int D, int KV, int R>
__global__ void __launch_bounds__(256) k_append(AppendP p) {
    constexpr int L = D / 8;          // lanes of a head
    constexpr int UPB = 256 / L;      // heads a workgroup takes at a time
    constexpr int PD = D + 4;
    __shared__ __attribute__((aligned(16))) float rowv[2][R][PD];
    __shared__ int s_page[R], s_tok[R], s_run[R];
    __shared__ float s_inv[2][R][D / 32];
    const int tid = threadIdx.x, j = tid % L, u = tid / L;
    int oa, ob;
    const bool turn = quad_offsets(p, j, oa, ob);

    if ((int)blockIdx.x >= p.kv_blocks) {  // queries
        const int64_t unit = (int64_t)(blockIdx.x - p.kv_blocks) * UPB + u;
        const int row = (int)(unit / p.q_heads), h = (int)(unit % p.q_heads);
        if (row >= p.rows) return;  // all lanes of a head together
        const float* src = p.x[0] + row * p.ld[0] + (size_t)h * D;
        f32x4 a = *(const f32x4*)(src + oa), b = *(const f32x4*)(src + ob);
        const int pos = p.pos[row];
        const bool live = pos >= 0 && pos < p.n_pos && (p.seq ? (unsigned)p.seq[row] < (unsigned)p.kv.n_seq : true);
        norm_turn<D>(p, p.w[0], turn && live, pos, oa, ob, j, a, b);
        if (!live) a = b = f32x4{0.f, 0.f, 0.f, 0.f};
        const size_t o = ((size_t)row * p.q_heads + h) * D;
        if (p.q_bf16) {
            uint16_t* q = (uint16_t*)p.q_out + o;
            *(u32x2*)(q + oa) = u32x2{f2bf2(a[0], a[1]), f2bf2(a[2], a[3])};
            *(u32x2*)(q + ob) = u32x2{f2bf2(b[0], b[1]), f2bf2(b[2], b[3])};
        } else {
            float* q = (float*)p.q_out + o;
            *(f32x4*)(q + oa) = a;
            *(f32x4*)(q + ob) = b;
        }
        return;
    }

    // keys and values: R rows of one head
    const KvView& kv = p.kv;
    const int h = blockIdx.x % kv.heads, r0 = (int)(blockIdx.x / kv.heads) * R;
    // rows 0..R-1 of keys, then of values, before the pages they go to are known
    constexpr int N = (2 * R + UPB - 1) / UPB;
    f32x4 xa[N], xb[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int i = u + e * UPB, which = i / R, row = r0 + i % R;
        xa[e] = xb[e] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (i < 2 * R && row < p.rows) {
            const float* src = p.x[1 + which] + row * p.ld[1 + which] + (size_t)h * D;
            xa[e] = *(const f32x4*)(src + oa);
            xb[e] = *(const f32x4*)(src + ob);
        }
    }
    if (tid < R) {
        const int row = r0 + tid;
        int page = -1, tok = -1;
        if (row < p.rows) {
            tok = p.pos[row];
            page = tok < p.n_pos ? kv_page(kv, p.seq ? p.seq[row] : 0, tok) : -1;
        }
        s_page[tid] = page;
        s_tok[tid] = page < 0 ? -1 : tok & (kv.P - 1);
    }
    __syncthreads();
    if (tid < R) {
        // 2: the first of 8 rows that are a whole unit of tokens, 1: a later one, 0: a row by itself
        int run = 0;
        for (int s = tid > 7 ? tid - 7 : 0; s <= tid; ++s) {
            if (s_page[s] < 0 || (s_tok[s] & 7) || s + 8 > R) continue;
            bool whole = true;
            for (int e = 1; e < 8; ++e) whole &= s_page[s + e] == s_page[s] && s_tok[s + e] == s_tok[s] + e;
            if (whole) run = s == tid ? 2 : 1;
        }
        s_run[tid] = run;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const int i = u + e * UPB, which = i / R, r = i % R;
        if (i >= 2 * R) break;
        if (which == 0) {
            const int pos = r0 + r < p.rows ? p.pos[r0 + r] : -1;
            norm_turn<D>(p, p.w[1], turn && pos >= 0 && pos < p.n_pos, pos, oa, ob, j, xa[e], xb[e]);
        }
        *(f32x4*)&rowv[which][r][oa] = xa[e];
        *(f32x4*)&rowv[which][r][ob] = xb[e];
    }
    __syncthreads();
    auto head_at = [&](int r) { return kv.pages + (size_t)s_page[r] * kv.page_bytes + (size_t)h * kv.head_bytes; };
    const int P = kv.P;
    if constexpr (KV == kKvBf16) {
        for (int i = tid; i < R * (D / 8); i += 256) {  // a key's 8 dims
            const int r = i % R, c = i / R;
            if (s_page[r] < 0) continue;
            const f32x4 a = *(const f32x4*)&rowv[0][r][8 * c], b = *(const f32x4*)&rowv[0][r][8 * c + 4];
            *(u32x4*)(head_at(r) + kv_k_unit(P, c, s_tok[r])) =
                u32x4{f2bf2(a[0], a[1]), f2bf2(a[2], a[3]), f2bf2(b[0], b[1]), f2bf2(b[2], b[3])};
        }
        for (int i = tid; i < R * D; i += 256) {  // a value's dim, of 8 tokens at once where they are a unit
            const int d = i % D, r = i / D;
            if (s_page[r] < 0 || s_run[r] == 1) continue;
            char* at = head_at(r) + kv_v_unit(P, D, s_tok[r] >> 3, d);
            if (s_run[r] == 2) {
                u32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = f2bf2(rowv[1][r + 2 * e][d], rowv[1][r + 2 * e + 1][d]);
                *(u32x4*)at = o;
            } else {
                ((uint16_t*)at)[s_tok[r] & 7] = f2bf(rowv[1][r][d]);
            }
        }
    } else {
        for (int i = tid; i < R * D / 16; i += 256) {  // scale of (key or value, row, 32 dims)
            const int r = i % R, c = i / R % (D / 32), which = i / (R * (D / 32));
            uint32_t amax = 0;  // the largest magnitude's bits: a NaN's are above all others
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const u32x4 x = *(const u32x4*)&rowv[which][r][32 * c + 4 * e];
#pragma unroll
                for (int k = 0; k < 4; ++k) amax = max(amax, x[k] & 0x7FFFFFFFu);
            }
            uint16_t bits;
            const float inv = scale_of(as_float(amax), bits);
            s_inv[which][r][c] = inv;
            if (s_page[r] >= 0)
                *(uint16_t*)(head_at(r) + (which ? kv_vs_off(P, D, c, s_tok[r]) : kv_ks_off(P, D, c, s_tok[r]))) = bits;
        }
        __syncthreads();
        for (int i = tid; i < R * (D / 16); i += 256) {  // a key's 16 codes: dims 64c + 8g.. and 64c + 32 + 8g..
            const int r = i % R, g = i / R % 4, c = i / (4 * R);
            if (s_page[r] < 0) continue;
            u32x4 o;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float inv = s_inv[0][r][2 * c + k];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f32x4 x = *(const f32x4*)&rowv[0][r][64 * c + 32 * k + 8 * g + 4 * q];
                    o[2 * k + q] = code_of(x[0], inv) | code_of(x[1], inv) << 8 | code_of(x[2], inv) << 16 | code_of(x[3], inv) << 24;
                }
            }
            *(u32x4*)(head_at(r) + kv_kq_unit(P, c, g, s_tok[r])) = o;
        }
        for (int i = tid; i < R * D / 2; i += 256) {  // dims 32c + m and 32c + 16 + m of a value
            const int m = i % 16, c = i / 16 % (D / 32), r = i / (D / 2);
            if (s_page[r] < 0 || s_run[r] == 1) continue;
            uint8_t* at = (uint8_t*)head_at(r) + kv_vq_unit(P, D, s_tok[r] >> 3, c, m);
            if (s_run[r] == 2) {
                u32x4 o = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float inv = s_inv[1][r + e][c];
                    o[e / 4] |= code_of(rowv[1][r + e][32 * c + m], inv) << (8 * (e % 4));
                    o[2 + e / 4] |= code_of(rowv[1][r + e][32 * c + 16 + m], inv) << (8 * (e % 4));
                }
                *(u32x4*)at = o;
            } else {
                const float inv = s_inv[1][r][c];
                at[s_tok[r] & 7] = (uint8_t)code_of(rowv[1][r][32 * c + m], inv);
                at[8 + (s_tok[r] & 7)] = (uint8_t)code_of(rowv[1][r][32 * c + 16 + m], inv);
            }
        }
    }
}

// a lane reads 8 dims of one cached row
template <int KV>
__global__ void __launch_bounds__(256) k_kv_read(KvView kv, const int32_t* seq, const int32_t* pos, int rows, uint16_t* k, uint16_t* v) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int c8 = kv.D / 8, c = (int)(i % c8), h = (int)(i / c8 % kv.heads);
    const int64_t r = i / c8 / kv.heads;
    if (r >= rows) return;
    const int P = kv.P, D = kv.D, page = kv_page(kv, seq ? seq[r] : 0, pos[r]), t = pos[r] & (P - 1);
    const char* at = kv.pages + (size_t)(page < 0 ? 0 : page) * kv.page_bytes + (size_t)h * kv.head_bytes;
    const size_t o = ((size_t)r * kv.heads + h) * D + 8 * c;
    u32x4 ok = {0, 0, 0, 0}, ov = ok;
    if (page >= 0) {
        if constexpr (KV == kKvBf16) {
            if (k) ok = *(const u32x4*)(at + kv_k_unit(P, c, t));
            if (v)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    ov[e / 2] |= (uint32_t)((const uint16_t*)(at + kv_v_unit(P, D, t >> 3, 8 * c + e)))[t & 7] << (16 * (e % 2));
        } else {
            if (k) {
                const int8_t* q = (const int8_t*)(at + kv_kq_unit(P, c / 8, c % 4, t)) + 8 * (c / 4 % 2);
                const float d = bf2f(*(const uint16_t*)(at + kv_ks_off(P, D, c / 4, t)));
#pragma unroll
                for (int e = 0; e < 4; ++e) ok[e] = f2bf2(q[2 * e] * d, q[2 * e + 1] * d);
            }
            if (v) {
                const float d = bf2f(*(const uint16_t*)(at + kv_vs_off(P, D, c / 4, t)));
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int dim = 8 * c + e;
                    x[e] = ((const int8_t*)(at + kv_vq_unit(P, D, t >> 3, dim / 32, dim % 16)))[dim / 16 % 2 * 8 + (t & 7)] * d;
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) ov[e] = f2bf2(x[2 * e], x[2 * e + 1]);
            }
        }
    }
    if (k) *(u32x4*)(k + o) = ok;
    if (v) *(u32x4*)(v + o) = ov;
}

template <int D, int KV>
hipError_t launch_append_of(AppendP p, hipStream_t st) {
    constexpr int upb = 256 / (D / 8);
    const int64_t qb = ((int64_t)p.rows * p.q_heads + upb - 1) / upb;
    // 16 rows of a head per workgroup make whole units of a prompt's values;
    // four end sooner where the GPU is not full (32 + 2 x 4 heads of 128, rows
    // of 16 / of 4 per workgroup: 1 row 4.8 / 4.0 us, 256 rows 7.4 / 4.8,
    // 2048 rows 14.1 / 16.5, 8192 rows 50 / 52)
    const bool few = p.rows <= kFewRows;
    p.kv_blocks = (p.rows + (few ? 3 : 15)) / (few ? 4 : 16) * p.kv.heads;
    const dim3 grid((uint32_t)(p.kv_blocks + qb));
    if (few)
        launch_kernel((k_append<D, KV, 4>), grid, dim3(256), 0, st, p);
    else
        launch_kernel((k_append<D, KV, 16>), grid, dim3(256), 0, st, p);
    return hipGetLastError();
}
}  // namespace

hipError_t launch_append(const KvView& kv, int type, const bq_append_args& a, hipStream_t st) {
    AppendP p;
    p.kv = kv;
    p.x[0] = a.q; p.x[1] = a.k; p.x[2] = a.v;
    p.ld[0] = a.ldq; p.ld[1] = a.ldk; p.ld[2] = a.ldv;
    p.w[0] = a.q_weight; p.w[1] = a.k_weight;
    p.pos = a.pos; p.seq = a.seq; p.rope = a.rope; p.q_out = a.q_out; p.eps = a.eps;
    p.rows = a.rows; p.q_heads = a.q_heads; p.rot = a.rot; p.n_pos = a.n_pos; p.interleaved = a.interleaved != 0;
    p.q_bf16 = a.q_type == BQ_TYPE_BF16;
    const bool q8 = type == kKvQ8;
    switch (kv.D) {
        case 64: return q8 ? launch_append_of<64, kKvQ8>(p, st) : launch_append_of<64, kKvBf16>(p, st);
        case 128: return q8 ? launch_append_of<128, kKvQ8>(p, st) : launch_append_of<128, kKvBf16>(p, st);
        default: return q8 ? launch_append_of<256, kKvQ8>(p, st) : launch_append_of<256, kKvBf16>(p, st);
    }
}

hipError_t launch_kv_read(const KvView& kv, int type, const int32_t* seq, const int32_t* pos, int rows, uint16_t* k, uint16_t* v,
                          hipStream_t st) {
    const int64_t n = (int64_t)rows * kv.heads * (kv.D / 8);
    const dim3 grid((uint32_t)((n + 255) / 256));
    if (type == kKvQ8)
        launch_kernel((k_kv_read<kKvQ8>), grid, dim3(256), 0, st, kv, seq, pos, rows, k, v);
    else
        launch_kernel((k_kv_read<kKvBf16>), grid, dim3(256), 0, st, kv, seq, pos, rows, k, v);
    return hipGetLastError();
}

}  // namespace bq
