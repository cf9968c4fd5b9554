// bq_sample.hip -- one token per row of logits: temperature, top-k, top-p,
// min-p, from a given uniform number.
//
// Kept tokens are a run of the row sorted by logit, so only the row's head has
// to be sorted.  Two launches:
//   k_sample_scan, one workgroup per 4096 logits: reads them once (the floor:
//     4 bytes a logit), keeps the head of its slice -- every logit not below a
//     threshold t, taken from the lanes' maxima in order, which leaves about 400
//     candidates for the whole row -- and, where no top-k bounds it, its sum of
//     exponentials.
//   k_sample_pick, one workgroup per row: takes the candidates not below the
//     largest t, which are the row's largest logits for sure, puts them in order
//     and cuts their running mass.  A cut that falls among them is exact.  Where it
//     does not (a flat row, hundreds of tokens kept, no filter and a draw behind
//     them), the row is read again, two or three times (struct Whole).
// Bounds: one row is latency, two launches and the pick's chain of loads, LDS
// and barriers (131072 logits 8.9 us: scan 3.9, pick 5); many rows the reading
// of the logits (64 rows of 131072 with top-p 15.8 us, 34 MB at 2.1 TB/s over both
// launches); a row read again 60 to 90 us.
// Slices are 256-logit blocks dealt in turn: likely tokens that lie together
// in the vocabulary spread over the slices.
// A mass is exp(x) in units of 2^-40 of the first token's, in 64-bit integers:
// the atomic sums come out the same in any order.  (The row's mass of the scan
// is a float sum per slice, in a fixed order.)
#include <algorithm>
#include <cmath>

#include "bq_device.hpp"
#include "bq_internal.hpp"

namespace bq {

namespace {
constexpr int kSlice = 4096;
constexpr int kMaxSlices = 256;
constexpr int kMaxCand = 1024;
constexpr int kWant = 384;  // candidates wanted of a row
typedef unsigned long long u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any logit

struct SliceInfo {
    u64 best;      // largest key
    float t;       // every logit >= t of the slice is a candidate (-inf: all finite ones, +inf: none)
    float sum;     // of exp((x - max) / temperature), where top-k does not bound the row
    int count, pad;
};

struct SampleP {
    const float* logits;
    int64_t ld;
    int vocab, slices, cap_log, rank;  // a slice has room for 2^cap_log candidates
    const float* temp;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* u;
    int32_t* out;
    SliceInfo* info;
    u64* cand;
};

// ordered bits of a logit (-0 as 0, NaN as -inf), and the sort key: larger
// logits first, then lower indices
BQ_DEV float clean(float x) { return x == x ? x + 0.f : -INFINITY; }
BQ_DEV uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
BQ_DEV float unordered(uint32_t o) { return as_float(o ^ (o >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
BQ_DEV u64 key_of(float x, int i) { return (u64)ordered(x) << 32 | (0xFFFFFFFFu - (uint32_t)i); }
BQ_DEV int index_of(u64 key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }
BQ_DEV u64 mass(float e) { return (u64)__builtin_rintf(e * 0x1p40f); }
BQ_DEV u64 shfl_xor64(u64 v, int d) {
    const uint32_t lo = __shfl_xor((uint32_t)v, d, 64), hi = __shfl_xor((uint32_t)(v >> 32), d, 64);
    return (u64)hi << 32 | lo;
}
// the wave's inclusive sums
template <int CTRL, int ROWS>
BQ_DEV u64 plus_dpp(u64 v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)v, CTRL, ROWS, 0xF, ROWS == 0xF);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(v >> 32), CTRL, ROWS, 0xF, ROWS == 0xF);
    return v + ((u64)hi << 32 | lo);
}
BQ_DEV int wave_scan32(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
}
BQ_DEV u64 wave_scan64(u64 v) {
    v = plus_dpp<0x111, 0xF>(v);   // row_shr:1
    v = plus_dpp<0x112, 0xF>(v);   // row_shr:2
    v = plus_dpp<0x114, 0xF>(v);   // row_shr:4
    v = plus_dpp<0x118, 0xF>(v);   // row_shr:8
    v = plus_dpp<0x142, 0xA>(v);   // row_bcast:15 into rows 1, 3
    return plus_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2, 3
}

// the value of lane ^ J (J < 64), without LDS
template <int J>
BQ_DEV uint32_t lane_xor(uint32_t v) {
    if constexpr (J == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, false);  // quad_perm [1,0,3,2]
    if constexpr (J == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, false);  // quad_perm [2,3,0,1]
    if constexpr (J == 4) {  // row_half_mirror is ^7, quad_perm [3,2,1,0] ^3
        return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, false), 0x1B, 0xF, 0xF, false);
    }
    if constexpr (J == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, false);  // row_ror:8
    if constexpr (J == 16) {  // both rows of a pair: [0] holds the even rows' values, [1] the odd rows'
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return threadIdx.x & 16 ? r[0] : r[1];
    }
    if constexpr (J == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return threadIdx.x & 32 ? r[0] : r[1];
    }
}
// one exchange of a bitonic network: the larger of the pair stays in the lower lane if `down`
template <int J>
BQ_DEV u64 exchange(u64 key, bool down) {
    const u64 o = (u64)lane_xor<J>((uint32_t)(key >> 32)) << 32 | lane_xor<J>((uint32_t)key);
    const bool larger = down == ((threadIdx.x & J) == 0);
    return larger == (o > key) ? o : key;
}

struct RowRule {
    float temp, top_p, min_p;
    int top_k;  // vocab: all
    bool greedy;
};
BQ_DEV RowRule rule_of(const SampleP& p, int row) {
    RowRule r;
    r.temp = p.temp ? p.temp[row] : 1.f;
    r.top_p = p.top_p ? p.top_p[row] : 1.f;
    r.min_p = p.min_p ? p.min_p[row] : 0.f;
    const int k = p.top_k ? p.top_k[row] : 0;
    r.top_k = k > 0 && k < p.vocab ? k : p.vocab;
    r.greedy = !(r.temp > 0.f) || r.top_k == 1;
    return r;
}

// the wave's maximum, in every lane
BQ_DEV float wave_max(float v) {
    v = fmaxf(v, dpp_f<0xB1, 0xF, true>(v));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp_f<0x4E, 0xF, true>(v));   // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp_f<0x141, 0xF, true>(v));  // row_half_mirror
    v = fmaxf(v, dpp_f<0x140, 0xF, true>(v));  // row_mirror
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

BQ_DEV u64 larger(u64 a, u64 b) { return a > b ? a : b; }
template <int J>
BQ_DEV u64 larger_xor(u64 v) {
    return larger(v, (u64)lane_xor<J>((uint32_t)(v >> 32)) << 32 | lane_xor<J>((uint32_t)v));
}
BQ_DEV u64 wave_max64(u64 v) {
    return larger_xor<32>(larger_xor<16>(larger_xor<8>(larger_xor<4>(larger_xor<2>(larger_xor<1>(v))))));
}

__global__ void __launch_bounds__(256) k_sample_scan(SampleP p) {
    constexpr int V = kSlice / 1024;  // 16-byte loads of a thread
    __shared__ float s_max[4], s_t[4], s_sum[4];
    __shared__ int s_count[4], s_at[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slice = blockIdx.x, row = blockIdx.y;
    const float* x = p.logits + (size_t)row * p.ld;
    // the slice's k-th run of four waves' blocks: block (4k + wave) * slices + slice
    float v[V][4];
    auto at = [&](int k) { return ((4 * k + wave) * p.slices + slice) * 256 + lane * 4; };
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int i = at(k);
        f32x4 a = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (i + 4 <= p.vocab) {
            a = *(const f32x4u*)(x + i);
        } else {
            for (int e = 0; e < 4; ++e)
                if (i + e < p.vocab) a[e] = x[i + e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = clean(a[e]);
    }
    const RowRule rule = rule_of(p, row);
    float mine = v[0][0];
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine = fmaxf(mine, v[k][e]);
    // the wave's threshold: the largest 16-bit prefix of the ordered bits that
    // more than `rank` of its lanes' maxima reach (a lower value than the
    // maximum itself is as good)
    uint32_t cut = 0;
    const uint32_t om = ordered(mine);
#pragma unroll
    for (int bit = 31; bit >= 16; --bit) {
        const uint32_t c = cut | 1u << bit;
        if (__popcll(__ballot(om >= c)) > p.rank) cut = c;
    }
    const float wmax = wave_max(mine);
    if (lane == 0) {
        s_t[wave] = cut < 0x00800000u ? -INFINITY : unordered(cut);  // below the lowest finite logit: all of them
        s_max[wave] = wmax;
    }
    __syncthreads();
    const float mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    // any threshold is right; the mean of the middle two is steadiest (one wave
    // may hold several of the row's likeliest tokens)
    const float t = 0.5f * fmaxf(fminf(s_t[0], s_t[1]), fminf(s_t[2], s_t[3])) +
                    0.5f * fminf(fmaxf(s_t[0], s_t[1]), fmaxf(s_t[2], s_t[3]));
    const float least = fmaxf(t, -3.402823466e38f);  // -inf is no candidate
    int count = 0, first = 0x7FFFFFFF;
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) count += __popcll(__ballot(v[k][e] >= least));
    if (__any(mine == mx)) {
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (v[k][e] == mx) first = min(first, at(k) + e);
        for (int d = 1; d < 64; d <<= 1) first = min(first, __shfl_xor(first, d, 64));
    }
    if (lane == 0) {
        s_count[wave] = count;
        s_at[wave] = first;
    }
    if (rule.top_k == p.vocab && !rule.greedy) {
        float sum = 0.f;
        if (mx > -INFINITY && mx < INFINITY) {
            const float inv = fminf(1.44269504088896341f / rule.temp, 3e38f);  // finite: 0 * inf is no mass
            if (inv > 0.f) {
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f((v[k][e] - mx) * inv);
            } else {  // an infinite temperature: the tokens above -inf
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += v[k][e] > -INFINITY ? 1.f : 0.f;
            }
        }
        sum = wave_sum_dpp63(sum);
        if (lane == 63) s_sum[wave] = sum;
    }
    __syncthreads();
    const int total = s_count[0] + s_count[1] + s_count[2] + s_count[3];
    const bool over = total > 1 << p.cap_log;
    if (!over && !rule.greedy) {
        u64* cand = p.cand + (((size_t)row * p.slices + slice) << p.cap_log);
        for (int w = 0; w < wave; ++w) cand += s_count[w];
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool in = v[k][e] >= least;
                const u64 mask = __ballot(in);
                if (mask == 0) continue;
                if (in) cand[__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] =
                    key_of(v[k][e], at(k) + e);
                cand += __popcll(mask);
            }
    }
    if (tid == 0) {
        SliceInfo* info = p.info + (size_t)row * p.slices + slice;
        info->best = key_of(mx, min(min(s_at[0], s_at[1]), min(s_at[2], s_at[3])));
        info->t = over ? INFINITY : t;
        info->sum = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
        info->count = over ? 0 : total;
    }
}

// exclusive scan over the workgroup's 1024 threads, and the total
BQ_DEV u64 scan1024(u64 v, u64* red, u64& total) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const u64 s = wave_scan64(v);
    __syncthreads();
    if (lane == 63) red[w] = s;
    __syncthreads();
    u64 before = 0;
    total = 0;
    for (int i = 0; i < 16; ++i) {
        if (i < w) before += red[i];
        total += red[i];
    }
    return before + s - v;
}

// bitonic sort, descending, of one key per thread; keys past thread n - 1 (a
// power of two >= 64) are zeros
BQ_DEV u64 sort_keys(u64 key, int n, u64* s_key) {
    const int tid = threadIdx.x;
    int turn = 0;
    __syncthreads();
    for (int k = 2; k <= n; k <<= 1) {
        const bool down = (tid & k) == 0;
        for (int j = k >> 1; j >= 64; j >>= 1) {
            // two buffers in turn: one barrier an exchange
            u64* at = s_key + (turn ^= 1) * kMaxCand;
            at[tid] = key;
            __syncthreads();
            const u64 o = at[tid ^ j];
            const bool larger = down == ((tid & j) == 0);
            key = larger == (o > key) ? o : key;
        }
        if (tid >= n) continue;  // whole waves
        if (k >= 64) key = exchange<32>(key, down);
        if (k >= 32) key = exchange<16>(key, down);
        if (k >= 16) key = exchange<8>(key, down);
        if (k >= 8) key = exchange<4>(key, down);
        if (k >= 4) key = exchange<2>(key, down);
        key = exchange<1>(key, down);
    }
    return key;
}

// The whole row.  A cut is found in two readings: the weights (1 each, or the
// masses) in 2048 even bins between the first logit and the last one whose mass
// counts, then the keys of the bin that the cut falls into, sorted.  Where one
// bin holds more than 1024 keys (many equal logits), by radix selection on the
// ordered bits of the logit, then of the index.
struct Whole {
    const float* x;
    int vocab;
    float mx, to_log2, per_bin;  // log2(e) / temperature; bins per unit of logit
    u64* bins;   // [2048]
    u64* keys;   // [2 kMaxCand]
    u64* red;    // [16]
    u64* found;  // [3]

    // f(key, logit) over the logits above -inf
    template <typename F>
    BQ_DEV void each(F f) const {
        constexpr int N = 4;  // loads in flight
        for (int i0 = 4 * threadIdx.x; i0 < vocab; i0 += 4096 * N) {
            f32x4 a[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const int i = i0 + 4096 * k;
                a[k] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (i + 4 <= vocab) {
                    a[k] = *(const f32x4u*)(x + i);
                } else {
                    for (int e = 0; e < 4; ++e)
                        if (i + e < vocab) a[k][e] = x[i + e];
                }
            }
#pragma unroll
            for (int k = 0; k < N; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float v = clean(a[k][e]);
                    if (v > -INFINITY) f(key_of(v, i0 + 4096 * k + e), v);
                }
        }
    }
    BQ_DEV u64 mass_of(float v) const { return mass(__builtin_amdgcn_exp2f((v - mx) * to_log2)); }
    BQ_DEV u64 weight(bool by_count, float v) const { return by_count ? 1 : mass_of(v); }
    BQ_DEV int bin_of(float v) const { return (int)fminf((mx - v) * per_bin, 2047.f); }  // rises as v falls

    // weights of the keys >= low into the bins
    BQ_DEV void fill(bool by_count, u64 low) const {
        __syncthreads();
        for (int i = threadIdx.x; i < 2048; i += 1024) bins[i] = 0;
        __syncthreads();
        each([&](u64 key, float v) {
            if (key < low) return;
            const u64 w = weight(by_count, v);
            if (w) atomicAdd(&bins[bin_of(v)], w);
        });
        __syncthreads();
    }
    BQ_DEV u64 filled() const {  // their sum
        u64 total;
        scan1024(bins[2 * threadIdx.x] + bins[2 * threadIdx.x + 1], red, total);
        return total;
    }

    // With the bins filled from the same keys: the first key in descending
    // order whose running weight meets w >= target (or w > target), and that
    // weight.  0 if none does; `many` where the bin holds too many.
    BQ_DEV u64 locate(bool by_count, double target, bool strict, u64 low, u64& upto, bool& many) const {
        const int tid = threadIdx.x;
        auto meets = [&](u64 w) { return strict ? (double)w > target : (double)w >= target; };
        __syncthreads();  // found[] of a call before has been read by every wave
        if (tid == 0) found[0] = ~0ull, found[2] = 0;
        __syncthreads();
        const u64 a = bins[2 * tid], b = bins[2 * tid + 1];
        u64 total;
        const u64 ex = scan1024(a + b, red, total);
        if (a && !meets(ex) && meets(ex + a)) {
            found[0] = 2 * tid;
            found[1] = ex;
        } else if (b && !meets(ex + a) && meets(ex + a + b)) {
            found[0] = 2 * tid + 1;
            found[1] = ex + a;
        }
        __syncthreads();
        const u64 bin = found[0], before = found[1];
        if (bin == ~0ull) return 0;
        each([&](u64 key, float v) {
            if (key < low || bin_of(v) != (int)bin) return;
            const u64 c = atomicAdd(&found[2], 1ull);
            if (c < kMaxCand) keys[c] = key;
        });
        __syncthreads();
        const int count = (int)found[2];
        if (count > kMaxCand) {
            many = true;
            return 0;
        }
        int n = 64;
        while (n < count) n <<= 1;
        u64 key = tid < count ? keys[tid] : 0;
        key = sort_keys(key, n, keys);
        const u64 w = tid < count ? weight(by_count, unordered((uint32_t)(key >> 32))) : 0;
        const u64 at = before + scan1024(w, red, total);
        if (tid == 0) found[0] = 0;
        __syncthreads();
        if (w && !meets(at) && meets(at + w)) {
            found[0] = key;
            found[1] = at + w;
        }
        __syncthreads();
        upto = found[1];
        return found[0];
    }

    // the same by radix selection
    BQ_DEV u64 select(bool by_count, double target, bool strict, u64 low) const {
        constexpr int kShift[6] = {53, 42, 32, 21, 10, 0}, kBits[6] = {11, 11, 10, 11, 11, 10};
        u64 prefix = 0;   // the digits found so far, in place
        u64 before = 0;   // the weight of larger keys
        for (int d = 0; d < 6; ++d) {
            const int sh = kShift[d], nb = 1 << kBits[d];
            __syncthreads();
            for (int i = threadIdx.x; i < 2048; i += 1024) bins[i] = 0;
            if (threadIdx.x == 0) found[0] = ~0ull;
            __syncthreads();
            each([&](u64 key, float v) {
                if (key < low || (d && (key ^ prefix) >> (sh + kBits[d]))) return;
                const u64 w = weight(by_count, v);
                if (w) atomicAdd(&bins[(key >> sh) & (nb - 1)], w);
            });
            __syncthreads();
            // thread i owns the i-th and (i + 1)-th bins from the top
            const int hi = nb - 1 - 2 * (int)threadIdx.x;
            const u64 a = hi >= 1 ? bins[hi] : 0, b = hi >= 1 ? bins[hi - 1] : 0;
            u64 total;
            const u64 ex = before + scan1024(a + b, red, total);
            auto meets = [&](u64 w) { return strict ? (double)w > target : (double)w >= target; };
            if (a && !meets(ex) && meets(ex + a)) {
                found[0] = hi;
                found[1] = ex;
            } else if (b && !meets(ex + a) && meets(ex + a + b)) {
                found[0] = hi - 1;
                found[1] = ex + a;
            }
            __syncthreads();
            if (found[0] == ~0ull) return 0;
            prefix |= found[0] << sh;
            before = found[1];
        }
        return prefix;
    }
    // either; bins must be filled from the keys >= low
    BQ_DEV u64 cut(bool by_count, double target, bool strict, u64 low, u64& upto) const {
        bool many = false;
        u64 key = per_bin > 0.f ? locate(by_count, target, strict, low, upto, many) : 0;
        if (many || !(per_bin > 0.f)) {
            key = select(by_count, target, strict, low);
            fill(by_count, low);  // it used the bins
            if (key && !by_count) upto = mass_from(key);
        }
        return key;
    }

    BQ_DEV u64 mass_from(u64 low) const {
        u64 s = 0, total;
        each([&](u64 key, float v) {
            if (key >= low) s += mass_of(v);
        });
        scan1024(s, red, total);
        return total;
    }
};

// The token of a row whose largest logits are sorted, by one wave: its lanes
// have E each, key[] and masses weight[] in descending order, `total` of them,
// all not below t.  -1: the cut may lie behind them.
constexpr u64 kBelow = 1ull << 63;  // of a weight: its token is less likely than min_p allows
template <int E>
BQ_DEV int decide(const SampleP& p, const RowRule& rule, const u64* key, u64* weight, int total, float mx, float t, double row_mass,
                  double u) {
    const int i0 = threadIdx.x * E;
    constexpr int kNone = kMaxCand + 1;
    u64 upto[E], sum = 0;
    int below = kNone;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
        const u64 w = weight[i0 + e];
        upto[e] = w & ~kBelow;
        if (w & kBelow) below = i0 + e;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) upto[e] = sum += upto[e];
    const u64 before = wave_scan64(sum) - sum;
#pragma unroll
    for (int e = 0; e < E; ++e) weight[i0 + e] = upto[e] += before;  // read by the other lanes
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const double all = (double)weight[total - 1];
    // mass of the first top_k; where t cuts them off, its bounds: the others
    // have at most the mass of a logit t each
    const bool whole = !(t > -INFINITY), cuts = rule.top_p < 1.f;
    const float e_t = expf((t - mx) / rule.temp);
    double z = rule.top_k <= total ? (double)weight[rule.top_k - 1] : whole ? all : row_mass, z_most = z;
    if (rule.top_k > total && !whole && rule.top_k < p.vocab) {
        z = all;
        z_most = all + (double)(rule.top_k - total) * (double)mass(e_t);
    }
    const double cut = (double)rule.top_p * z, cut_most = (double)rule.top_p * z_most;
    // the first index that a rule shuts out, with either
    auto first_of = [&](int mine) {
        const u64 any = __ballot(mine < kNone);
        return any ? __builtin_amdgcn_readlane(mine, __builtin_ctzll(any)) : kNone;
    };
    int stop = kNone, stop_most = kNone;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
        const int i = i0 + e;
        if (i == 0 || i >= total) continue;
        const double ex = (double)(e ? upto[e - 1] : before);
        if (i >= rule.top_k || i >= below || (cuts && ex >= cut)) stop = i;
        if (i >= rule.top_k || i >= below || (cuts && ex >= cut_most)) stop_most = i;
    }
    int kept = first_of(stop), kept_most = first_of(stop_most);
    const bool end = whole || total >= rule.top_k || e_t < rule.min_p;  // nothing behind them is kept
    if (kept == kNone && (end || (cuts && all >= cut))) kept = total;
    if (kept_most == kNone && (end || (cuts && all >= cut_most))) kept_most = total;
    double target = u * row_mass;
    if (kept == kNone && rule.top_k == p.vocab && !cuts && !(rule.min_p > 0.f) && target < all) {
        kept = total;  // the whole row is kept, and the draw falls among these
    } else {
        if (kept == kNone || kept != kept_most) return -1;
        target = u * (double)weight[kept - 1];
    }
    int at = kNone;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
        const int i = i0 + e;
        if (i < kept && ((double)upto[e] > target || i == kept - 1)) at = i;
    }
    return index_of(key[first_of(at)]);
}

constexpr int kBins = 1024, kManyKeys = 32;
__global__ void __launch_bounds__(1024) k_sample_pick(SampleP p) {
    __shared__ u64 s_key[2 * kMaxCand], s_bins[2048], s_red[16], s_found[3];
    __shared__ int s_count[kMaxSlices], s_sum[16], s_total, s_pick, s_many;
    __shared__ u64 s_best;
    __shared__ float s_t, s_least[16];
    const int tid = threadIdx.x, row = blockIdx.x;
    const RowRule rule = rule_of(p, row);
    const double u = (double)p.u[row];
    const SliceInfo* info = p.info + (size_t)row * p.slices;
    // two slots a thread are read beside the counts that say which of them hold
    // a candidate: all of them up to 32 slices
    const int slots = p.slices << p.cap_log;
    const u64* cand = p.cand + (size_t)row * slots;
    u64 k0 = tid < slots ? cand[tid] : 0, k1 = tid + 1024 < slots ? cand[tid + 1024] : 0;
    int *const count = (int*)s_bins, *const start = count + kBins;  // of a bin's keys
    count[tid] = 0;
    double row_mass = 0;  // wave 0's
    if (tid < 64) {
        // four slices a lane: the largest key, the largest threshold, the mass
        constexpr int N = kMaxSlices / 64;
        SliceInfo in[N];
        u64 best = 0;
        float t = -INFINITY;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            in[i] = SliceInfo{0, -INFINITY, 0.f, 0, 0};
            if (64 * i + tid < p.slices) in[i] = info[64 * i + tid];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (64 * i + tid < p.slices) s_count[64 * i + tid] = in[i].count;
            best = larger(best, in[i].best);
            t = fmaxf(t, in[i].t);
        }
        best = wave_max64(best);
        t = wave_max(t);
        if (rule.top_k == p.vocab) {
            const float mx = unordered((uint32_t)(best >> 32));
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (in[i].sum > 0.f)
                    row_mass += (double)in[i].sum * (double)expf((unordered((uint32_t)(in[i].best >> 32)) - mx) / rule.temp);
            for (int d = 1; d < 64; d <<= 1) row_mass += __shfl_xor(row_mass, d, 64);
            row_mass *= 0x1p40;
        }
        if (tid == 0) {
            s_best = best;
            s_t = t;
            s_total = s_many = 0;
        }
    }
    __syncthreads();
    const float mx = unordered((uint32_t)(s_best >> 32));
    if (rule.greedy || !(mx > -INFINITY) || mx == INFINITY) {
        // a row of -inf has its largest key at index 0
        if (tid == 0) p.out[row] = index_of(s_best);
        return;
    }
    // the candidates not below t, the row's largest logits for sure (in any order: they are sorted)
    const float t = s_t;
    const uint32_t least = ordered(t);
    auto sure = [&](int at, u64 key) {
        return at < slots && (at & ((1 << p.cap_log) - 1)) < s_count[at >> p.cap_log] && (uint32_t)(key >> 32) >= least;
    };
    bool in0 = sure(tid, k0), in1 = sure(tid + 1024, k1);
    int lost = 0;
    if (slots > 2048) {  // packed: one a thread
        auto take = [&](bool is, u64 key) {
            const u64 mask = __ballot(is);
            if (mask == 0) return;
            int to = 0;
            if ((tid & 63) == 0) to = atomicAdd(&s_total, __popcll(mask));
            to = __builtin_amdgcn_readfirstlane(to) +
                 __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
            if (is && to < kMaxCand) s_key[to] = key;
        };
        take(in0, k0);
        take(in1, k1);
        for (int at = tid + 2048; at - tid < slots; at += 2048) {
            const u64 a = at < slots ? cand[at] : 0, b = at + 1024 < slots ? cand[at + 1024] : 0;
            take(sure(at, a), a);
            take(sure(at + 1024, b), b);
        }
        __syncthreads();
        lost = max(0, s_total - kMaxCand);
        in0 = tid < s_total;
        in1 = false;
        if (in0) k0 = s_key[tid];
    }
    // Sorted by bins of their distance to t, even in its logarithm (most lie
    // near t): a key's place is where its bin starts plus its larger ones there.
    const float per = 1.f / (mx - t);
    const bool even = t > -INFINITY && per > 0.f && per < INFINITY;
    auto bin_of = [&](u64 key) {  // of the least key: 0x382
        const float d = (unordered((uint32_t)(key >> 32)) - t) * per + 0x1p-7f;
        return even ? 0x382 - min(max((__builtin_bit_cast(int, d) - 0x3C000000) >> 16, 0), 0x382) : 0;
    };
    const int b0 = in0 ? bin_of(k0) : 0, b1 = in1 ? bin_of(k1) : 0;
    const int at0 = in0 ? atomicAdd(&count[b0], 1) : 0, at1 = in1 ? atomicAdd(&count[b1], 1) : 0;
    __syncthreads();
    {
        const int c = count[tid], w = tid >> 6;
        const int upto = wave_scan32(c);
        if ((tid & 63) == 63) s_sum[w] = upto;
        if (c > kManyKeys) s_many = 1;
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            before += i < w ? s_sum[i] : 0;
            all += s_sum[i];
        }
        start[tid] = before + upto - c;
        if (tid == 0) s_total = all + lost;
        __syncthreads();
    }
    const int total = s_total;
    if (total > 0 && total <= kMaxCand) {
        if (in0) s_key[start[b0] + at0] = k0;
        if (in1) s_key[start[b1] + at1] = k1;
        __syncthreads();
        int n = 64;
        while (n < total) n <<= 1;
        u64 *const keys = s_key + kMaxCand, *const weights = s_bins + kMaxCand;
        u64 key = tid < total ? s_key[tid] : 0;
        int to = tid;
        if (s_many) {
            key = sort_keys(key, n, s_key);
            __syncthreads();
        } else if (tid < total) {
            const int b = bin_of(key), c = count[b], from = start[b];
            to = from;
            for (int i = 0; i < c; ++i) to += s_key[from + i] > key;
        }
        if (tid < n) {
            const float e = tid < total ? expf((unordered((uint32_t)(key >> 32)) - mx) / rule.temp) : 0.f;
            keys[to] = key;
            weights[to] = mass(e) | (e < rule.min_p ? kBelow : 0);
        }
        __syncthreads();
        if (tid < 64) {
            int pick;
            if (n == 64) pick = decide<1>(p, rule, keys, weights, total, mx, t, row_mass, u);
            else if (n == 128) pick = decide<2>(p, rule, keys, weights, total, mx, t, row_mass, u);
            else if (n == 256) pick = decide<4>(p, rule, keys, weights, total, mx, t, row_mass, u);
            else if (n == 512) pick = decide<8>(p, rule, keys, weights, total, mx, t, row_mass, u);
            else pick = decide<16>(p, rule, keys, weights, total, mx, t, row_mass, u);
            if (tid == 0) {
                s_pick = pick;
                if (pick >= 0) p.out[row] = pick;
            }
        }
        __syncthreads();
        if (s_pick >= 0) return;
    }
    // the head was not enough: the whole row
    Whole r{p.logits + (size_t)row * p.ld, p.vocab, mx, fminf(1.44269504088896341f / rule.temp, 3e38f), 0.f, s_bins, s_key, s_red, s_found};
    float last = INFINITY;
    r.each([&](u64, float v) { last = fminf(last, v); });
    last = -wave_max(-last);
    if ((tid & 63) == 0) s_least[tid >> 6] = last;
    __syncthreads();
    for (int i = 0; i < 16; ++i) last = fminf(last, s_least[i]);
    const float range = fminf(mx - last, 32.f * rule.temp);  // e^-32 is below half a unit of mass
    r.per_bin = range > 0.f ? 2047.f / range : 0.f;
    u64 low = 0, kept = 0;  // the keys kept are >= low, of mass `kept`
    if (rule.top_k < p.vocab) {
        r.fill(true, 0);
        low = r.cut(true, (double)rule.top_k, false, 0, kept);  // 0: fewer finite ones
    }
    r.fill(false, low);
    kept = r.filled();
    // from here on only the kept mass changes: the bins serve every cut
    const u64 from = low;
    if (rule.top_p < 1.f) {
        u64 upto = 0;
        const u64 at = rule.top_p > 0.f ? r.cut(false, (double)rule.top_p * (double)kept, false, from, upto) : s_best;
        if (!(rule.top_p > 0.f)) upto = mass(1.f);
        if (at) low = at, kept = upto;
    }
    if (rule.min_p > 0.f) {
        // the smallest key whose weight is at least min_p: weights fall with the key
        u64 least = s_best;
        r.each([&](u64 key, float v) {
            if (key < least && expf((v - mx) / rule.temp) >= rule.min_p) least = key;
        });
        for (int d = 1; d < 64; d <<= 1) {
            const u64 o = shfl_xor64(least, d);
            least = o < least ? o : least;
        }
        __syncthreads();
        if ((tid & 63) == 0) s_red[tid >> 6] = least;
        __syncthreads();
        for (int i = 0; i < 16; ++i) least = s_red[i] < least ? s_red[i] : least;
        if (least > low) low = least, kept = r.mass_from(low);
    }
    u64 upto;
    u64 pick = r.cut(false, u * (double)kept, true, from, upto);
    if (pick < low) pick = r.cut(false, (double)kept, false, from, upto);  // u = 1: the last kept key with a mass
    if (tid == 0) p.out[row] = pick ? index_of(pick) : index_of(s_best);
}

int slices_of(int vocab) { return (vocab + kSlice - 1) / kSlice; }
// room for a slice's candidates: 64, or three times those wanted of it, so that
// few rows have a slice that overflows
int cap_log_of(int slices) {
    int n = 6;
    while (1 << n < std::min(kMaxCand, 3 * kWant / slices)) ++n;
    return n;
}
}  // namespace

size_t sample_work_bytes(int rows, int vocab) {
    const int s = slices_of(vocab);
    return (size_t)rows * s * (sizeof(SliceInfo) + (sizeof(u64) << cap_log_of(s)));
}

hipError_t launch_sample(const float* logits, int64_t ld, int rows, int vocab, const float* temp, const int32_t* top_k,
                         const float* top_p, const float* min_p, const float* u, int32_t* out, void* work, hipStream_t st) {
    SampleP p;
    p.logits = logits; p.ld = ld; p.vocab = vocab;
    p.slices = slices_of(vocab);
    p.cap_log = cap_log_of(p.slices);
    // each wave's threshold is one of its 64 lanes' maxima of 16 logits: the
    // rank-th leaves about 64 ln(64 / (64 - rank)) of its 1024 above it
    p.rank = std::max(2, std::min(62, (int)(64 * (1 - std::exp(-(double)kWant / p.slices / 256)))));
    p.temp = temp; p.top_k = top_k; p.top_p = top_p; p.min_p = min_p; p.u = u; p.out = out;
    p.info = (SliceInfo*)work;
    p.cand = (u64*)(p.info + (size_t)rows * p.slices);
    launch_kernel(k_sample_scan, dim3(p.slices, rows), dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    launch_kernel(k_sample_pick, dim3(rows), dim3(1024), 0, st, p);
    return hipGetLastError();
}

}  // namespace bq
