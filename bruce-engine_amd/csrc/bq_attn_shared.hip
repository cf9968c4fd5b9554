// bq_attn_shared.hip -- attention of 1..8 new tokens per sequence, for sequences in
// groups that share a long prefix.
//
//   o = sum_j 2^(x_j - m) v_j / sum_j 2^(x_j - m),  x_j = scale log2(e) q.k_j
// The sum over a group's prefix is taken for the query rows of all its sequences
// together, so the prefix' K and V are read once per row tile instead of once per
// sequence; the sum over a sequence's own tokens for its rows alone (bq_attn.hip's
// scheme in both).  Sums and maxima of the two, and of the pieces that each is cut
// into, go to the workspace; a second launch joins them in their order.
#include <algorithm>

#include "bq_attn_dev.hpp"
#include "bq_internal.hpp"

namespace bq {

namespace {
struct SharedP {
    KvView kv;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    const int32_t* kv_len;
    const int32_t* group0;
    const int32_t* prefix;
    float* part;      // [pieces][n_rows][q_heads][D], the prefix' pieces first, then [..][2] (m, l)
    int64_t ml;       // floats before the (m, l) part
    int n_groups, max_prefix;
    int rows, n_rows, q_heads, G, max_len, window, sinks, q_bf16, out_bf16;
    int ptiles, psplit, ttiles, tsplit;  // row tiles per head and pieces: of the prefixes, of a sequence's own tokens
    float scale;      // scale * log2(e)
};

BQ_DEV int length_of(const SharedP& p, int seq) {
    return min(max(p.kv_len[seq], 0), min(p.max_len, p.kv.max_pages << p.kv.plog));
}
BQ_DEV int prefix_of(const SharedP& p, int g) {
    return min(max(p.prefix[g], 0), min(p.max_prefix, p.kv.max_pages << p.kv.plog));
}
// sequences [s0, s1) of a group, inside the batch whatever group0 holds
BQ_DEV void group_of(const SharedP& p, int g, int& s0, int& s1) {
    s0 = min(max(p.group0[g], 0), p.kv.n_seq);
    s1 = min(max(p.group0[g + 1], s0), p.kv.n_seq);
}
// the group that holds a sequence, -1: none (the same in every lane of a wave)
BQ_DEV int group_with(const SharedP& p, int seq) {
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 < p.n_groups; g0 += 64) {
        int s0 = 0, s1 = 0;
        if (g0 + lane < p.n_groups) group_of(p, g0 + lane, s0, s1);
        const uint64_t in = __ballot(seq >= s0 && seq < s1);
        if (in) return g0 + __builtin_ctzll(in);
    }
    return -1;
}
// the group whose row tiles (of T query rows) include the tile-th of all, and its
// number among them; -1: there are fewer
template <int T>
BQ_DEV int tile_group(const SharedP& p, int& tile) {
    const int lane = threadIdx.x & 63, per = p.rows * p.G;
    for (int g0 = 0; g0 < p.n_groups; g0 += 64) {
        int s0 = 0, s1 = 0;
        if (g0 + lane < p.n_groups) group_of(p, g0 + lane, s0, s1);
        const int n = ((s1 - s0) * per + T - 1) / T;
        int upto = n;
        for (int d = 1; d < 64; d <<= 1) {
            const int below = __shfl_up(upto, d, 64);
            if (lane >= d) upto += below;
        }
        const uint64_t past = __ballot(upto > tile);
        if (past) {
            const int at = __builtin_ctzll(past);
            tile -= __builtin_amdgcn_readlane(upto - n, at);
            return g0 + at;
        }
        tile -= __builtin_amdgcn_readlane(upto, 63);
    }
    return -1;
}

// the steps of tokens from .. upto - 1 that rows at positions pfirst..plast see
BQ_DEV Steps steps_of(const SharedP& p, int pfirst, int plast, int from, int upto) {
    Steps s;
    const int stop = (min(upto, plast + 1) + 31) >> 5;
    s.b = from >> 5;
    s.lo = p.window ? max(0, pfirst - p.window + 1) : 0;
    s.lo_step = max(s.lo >> 5, s.b);
    s.ns = p.window ? max(0, min(min(s.lo_step, (p.sinks + 31) >> 5), stop) - s.b) : 0;
    s.n = min(upto, plast + 1) <= from ? 0 : s.ns + max(0, stop - s.lo_step);
    return s;
}

BQ_DEV void store4(const SharedP& p, size_t at, f32x4 a) {
    if (p.out_bf16)
        *(u32x2*)((uint16_t*)p.out + at) = u32x2{f2bf2(a[0], a[1]), f2bf2(a[2], a[3])};
    else
        *(f32x4*)((float*)p.out + at) = a;
}

// NQ parts of q, NP of a softmax weight
template <int D, int KV, int NQ, int NP>
__global__ void __launch_bounds__(256, D <= 128 ? 2 : 1) k_attn_shared(SharedP p) {
    constexpr int KS = D / 32, DT = D / 16;
    constexpr bool CUT = true;
    __shared__ int s_page[kRound * 2];
    __shared__ __attribute__((aligned(16))) float s_o[kWaves][16][D + 4];
    __shared__ float s_m[kWaves][16], s_l[kWaves][16], s_mt[16], s_lt[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const KvView& kv = p.kv;
    // the prefixes' workgroups first, then the sequences' own
    int u = blockIdx.x, seq, h, tile, split, nsplit, from, upto, M, piece0;
    const bool shared = u < p.ptiles * kv.heads * p.psplit;
    if (shared) {
        tile = u % p.ptiles;
        h = u / p.ptiles % kv.heads;
        split = u / (p.ptiles * kv.heads);
        nsplit = p.psplit;
        piece0 = 0;
        const int gr = tile_group<16>(p, tile);
        if (gr < 0) return;
        int s1;
        group_of(p, gr, seq, s1);
        M = (s1 - seq) * p.rows * p.G;
        from = 0;
        upto = prefix_of(p, gr);
        if (tile < 0 || tile > (M - 1) / 16) return;  // group0 is not what it should be
    } else {
        u -= p.ptiles * kv.heads * p.psplit;
        split = u % p.tsplit;
        u /= p.tsplit;
        h = u % kv.heads;
        tile = u / kv.heads % p.ttiles;
        seq = u / (kv.heads * p.ttiles);
        nsplit = p.tsplit;
        piece0 = p.psplit;
        M = p.rows * p.G;
        const int gr = group_with(p, seq);
        from = gr < 0 ? 0 : prefix_of(p, gr);
        upto = 0x7FFFFFFF;
    }
    // the lane's query row: of sequence seq + rs its new token i, head r % G of the group
    const int first = tile * 16, last = min(M, first + 16) - 1, r = min(first + c, last);
    const int rs = r / (p.rows * p.G), i = r / p.G % p.rows;
    const int pos = length_of(p, seq + rs) - p.rows + i;
    int pfirst = pos, plast = pos;
    for (int d = 1; d < 16; d <<= 1) {
        pfirst = min(pfirst, __shfl_xor(pfirst, d, 64));
        plast = max(plast, __shfl_xor(plast, d, 64));
    }
    pfirst = __builtin_amdgcn_readfirstlane(pfirst);
    plast = __builtin_amdgcn_readfirstlane(plast);
    const size_t qat = (size_t)(seq * p.rows + r / p.G) * p.ldq + (size_t)(h * p.G + r % p.G) * D;
    const Steps st = steps_of(p, pfirst, plast, from, upto);
    const int end = plast + 1, lo = st.lo, n = st.n;
    const int per = (n + nsplit - 1) / nsplit;
    const int v0 = min(n, split * per), v1 = min(n, v0 + per);
#include "bq_attn_rows.inc"
    for (int e = tid; e < 16 * (D / 4); e += 256) {
        const int row = e / (D / 4), d = e % (D / 4) * 4, r = first + row;
        if (r > last) continue;
        const size_t at = ((size_t)(piece0 + split) * p.n_rows + seq * p.rows + r / p.G) * p.q_heads + h * p.G + r % p.G;
        if (d == 0) *(u32x2*)(p.part + p.ml + at * 2) = u32x2{__builtin_bit_cast(uint32_t, s_mt[row]), __builtin_bit_cast(uint32_t, s_lt[row])};
        if (v0 >= v1) continue;  // l is 0: the row is not read
        f32x4 a = *(const f32x4*)&s_o[0][row][d];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) a += *(const f32x4*)&s_o[w][row][d];
        *(f32x4*)(p.part + at * D + d) = a;
    }
}

// joins the pieces of one query row: D / 4 lanes per piece, the pieces dealt over the
// rest of the workgroup's lanes, in a fixed order
template <int D>
__global__ void __launch_bounds__(256) k_attn_shared_join(SharedP p) {
    constexpr int T = 256, L = D / 4, S = T / L;
    __shared__ __attribute__((aligned(16))) float s_o[S][D];
    __shared__ float s_l[S], s_mx[T / 64];
    const int tid = threadIdx.x, row = blockIdx.x / p.q_heads, head = blockIdx.x % p.q_heads;
    const int64_t rows = (int64_t)p.n_rows * p.q_heads;
    // a sequence of no group has no prefix pieces
    const int first = group_with(p, row / p.rows) < 0 ? p.psplit : 0, n = p.psplit + p.tsplit;
    const float* ml = p.part + p.ml + (int64_t)blockIdx.x * 2;
    float mt = kNone;
    for (int s = first + tid; s < n; s += T) mt = fmaxf(mt, ml[s * rows * 2]);
    for (int d = 1; d < 64; d <<= 1) mt = fmaxf(mt, __shfl_xor(mt, d, 64));
    if ((tid & 63) == 0) s_mx[tid >> 6] = mt;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < T / 64; ++w) mt = fmaxf(mt, s_mx[w]);
    f32x4 a = {0.f, 0.f, 0.f, 0.f};
    float lt = 0.f;
#pragma unroll 4
    for (int s = first + tid / L; s < n; s += S) {
        const float l = ml[s * rows * 2 + 1];
        if (l == 0.f) continue;  // nothing was stored
        const float f = __builtin_amdgcn_exp2f(ml[s * rows * 2] - mt);
        a += *(const f32x4*)(p.part + (s * rows + blockIdx.x) * D + tid % L * 4) * f;
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
    store4(p, (size_t)row * p.ldo + (size_t)head * D + tid * 4, lt == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : a * (1.f / lt));
}

template <int D, int KV>
hipError_t launch_of(const SharedP& p, hipStream_t st) {
    const uint32_t units = (uint32_t)(p.ptiles * p.kv.heads * p.psplit + p.kv.n_seq * p.ttiles * p.kv.heads * p.tsplit);
    if (p.q_bf16 && p.out_bf16)
        launch_kernel((k_attn_shared<D, KV, 1, 1>), dim3(units), dim3(256), 0, st, p);
    else
        launch_kernel((k_attn_shared<D, KV, KV == kKvQ8 ? 2 : 3, KV == kKvQ8 ? 2 : 3>), dim3(units), dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    launch_kernel((k_attn_shared_join<D>), dim3((uint32_t)(p.n_rows * p.q_heads)), dim3(256), 0, st, p);
    return hipGetLastError();
}
}  // namespace

// Row tiles of all groups together, per head: every group may end with a broken one.
static int64_t shared_tiles(int n_seq, int rows, int G, int n_groups) {
    return ((int64_t)n_seq * rows * G + 15) / 16 + std::min(n_groups, n_seq) - 1;
}

SharedPlan shared_plan(int type, int n_seq, int rows, int q_heads, int kv_heads, int D, int max_len, int n_groups, int max_prefix, int window,
                       int sinks, int cus) {
    SharedPlan s;
    const int G = q_heads / kv_heads;
    const int64_t tiles = shared_tiles(n_seq, rows, G, n_groups);
    const int64_t prefix = std::min<int64_t>(decode_reach(rows, window, sinks, max_len), max_prefix);
    const int64_t own = std::min<int64_t>(decode_reach(rows, window, sinks, max_len), std::max(max_len - max_prefix, 1));
    const int64_t each = ((prefix + 31) / 32 + kWaves - 1) / kWaves;
    s.ptiles = tiles;
    s.psplit = (int)std::max<int64_t>(1, std::min<int64_t>(each, 2 * cus / (tiles * kv_heads)));
    s.ttiles = (rows * G + 15) / 16;
    s.tsplit = decode_splits(type, n_seq, rows, q_heads, kv_heads, D, own, cus);
    return s;
}
size_t shared_part_floats(const SharedPlan& s, int n_rows, int q_heads, int D) {
    return (size_t)(s.psplit + s.tsplit) * n_rows * q_heads * (D + 2);
}

hipError_t launch_attn_shared(const KvView& kv, int type, const bq_attn_args& a, const bq_attn_prefix& x, const SharedPlan& s, hipStream_t st) {
    SharedP p;
    p.kv = kv;
    p.q = a.q; p.out = a.out; p.ldq = a.ldq; p.ldo = a.ldo; p.kv_len = a.kv_len;
    p.group0 = x.group0; p.prefix = x.len; p.n_groups = x.n_groups; p.max_prefix = x.max_len;
    p.rows = a.rows; p.n_rows = a.n_rows; p.q_heads = a.q_heads; p.G = a.q_heads / kv.heads;
    p.max_len = a.max_len; p.window = a.window; p.sinks = a.sinks;
    p.q_bf16 = a.q_type == BQ_TYPE_BF16; p.out_bf16 = a.out_type == BQ_TYPE_BF16;
    p.scale = a.scale * 1.44269504088896341f;
    p.ptiles = (int)s.ptiles; p.psplit = s.psplit; p.ttiles = s.ttiles; p.tsplit = s.tsplit;
    p.part = (float*)a.work;
    p.ml = (int64_t)(s.psplit + s.tsplit) * a.n_rows * a.q_heads * kv.D;
    const bool q8 = type == kKvQ8;
    switch (kv.D) {
        case 64: return q8 ? launch_of<64, kKvQ8>(p, st) : launch_of<64, kKvBf16>(p, st);
        case 128: return q8 ? launch_of<128, kKvQ8>(p, st) : launch_of<128, kKvBf16>(p, st);
        default: return q8 ? launch_of<256, kKvQ8>(p, st) : launch_of<256, kKvBf16>(p, st);
    }
}

}  // namespace bq
