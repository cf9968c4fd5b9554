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

#include "bq_attn_dev.hpp"
#include "bq_internal.hpp"

namespace bq {

namespace {
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

// the steps that a tile's rows at positions pfirst..plast see
BQ_DEV Steps steps_of(const DecodeP& p, int pfirst, int plast) {
    Steps s;
    s.b = 0;
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
    const size_t qat = (size_t)(seq * p.rows + i) * p.ldq + (size_t)(h * p.G + r % p.G) * D;
    const Steps st = steps_of(p, pfirst, plast);
    const int end = plast + 1, lo = st.lo, n = st.n;
    const int per = (n + p.nsplit - 1) / p.nsplit;
    const int v0 = min(n, (int)blockIdx.x * per), v1 = min(n, v0 + per);
    constexpr bool CUT = false;
    constexpr int from = 0, upto = 0;
#include "bq_attn_rows.inc"
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
