// bq_logprob.hip -- of rows of logits: log probability and rank of a given token,
// entropy, and the likeliest tokens with their log probabilities.
//
// With M the row's largest logit (its first), x = (logit - M) / T and r the sum of
// exp(x) over all tokens but that first one:
//   log p = x - log1p(r),  H = log1p(r) - sum exp(x) x / (1 + r)
// so neither cancels: a row that is nearly sure keeps r, and H, to fp32's relative
// precision.  Two launches:
//   k_logprob_scan, one workgroup per 4096 logits: reads them once (the floor: 4 bytes
//     a logit), and leaves the slice's largest, its two sums, its tokens that come
//     before the given one, and, for more than one alternative, its candidates: the
//     logits not below a threshold that at least `top` of the slice's reach, taken
//     from the lanes' maxima.  Where these are too many (equal logits), the slice's
//     `top` largest exactly, by bisection on the ordered bits, then on the index.
//   k_logprob_join, one workgroup per row: joins the slices in their order, and ranks
//     the candidates not below the largest threshold by counting.
#include <algorithm>
#include <cmath>

#include "bq_device.hpp"
#include "bq_internal.hpp"

namespace bq {

namespace {
constexpr int kSlice = 4096;
constexpr int kKeys = 1024;  // candidates that the join holds at once
constexpr int kStep = 768;   // and looks at between two counts of them
static_assert(kKeys - kStep >= 2 * BQ_MAX_TOP, "the likeliest so far and a step's candidates fit");
typedef unsigned long long u64;
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start at any logit

struct SliceInfo {
    u64 best;        // largest key
    float sum, dot;  // of 2^y and 2^y y over the slice but its first largest, y relative to that (log2)
    uint32_t t;      // ordered bits that at least `top` of the slice's logits reach (0: none known)
    int before, count, pad;
};

struct LogprobP {
    const float* logits;
    int64_t ld;
    int vocab, slices, cap_log, top;  // a slice has room for 2^cap_log candidates (top > 1)
    const float* temp;
    const int32_t* tokens;
    float* logprob;
    int32_t* rank;
    float* entropy;
    int32_t* top_tokens;
    float* top_logprobs;
    SliceInfo* info;
    u64* cand;
};

// ordered bits of a logit (-0 as 0, NaN as -inf), and the sort key: larger logits
// first, then lower indices
BQ_DEV float clean(float x) { return x == x ? x + 0.f : -INFINITY; }
BQ_DEV uint32_t ordered(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    return b ^ (b >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
BQ_DEV float unordered(uint32_t o) { return as_float(o ^ (o >> 31 ? 0x80000000u : 0xFFFFFFFFu)); }
BQ_DEV u64 key_of(float x, int i) { return (u64)ordered(x) << 32 | (0xFFFFFFFFu - (uint32_t)i); }
BQ_DEV int index_of(u64 key) { return (int)(0xFFFFFFFFu - (uint32_t)key); }
BQ_DEV float value_of(u64 key) { return unordered((uint32_t)(key >> 32)); }

// y = (v - m) log2(e) / T for v <= m, m finite, at least -1000 (2^-1000 is 0; so are the
// terms of -inf, whatever T is).  From T = 1 on a quarter of each is subtracted, which is
// exact and cannot overflow; below T = 2^-100 the difference is scaled up first, so that
// no factor is infinite.
struct Scaled {
    float q, up, mul;
    BQ_DEV explicit Scaled(float T) {
        q = T >= 1.f ? 0.25f : 1.f;
        up = T < 0x1p-100f ? 0x1p60f : 1.f;
        mul = 1.44269504088896341f / (T * q * up);
    }
    BQ_DEV float y(float v, float m) const { return fmaxf((v * q - m * q) * up * mul, -1000.f); }
};
// x = (v - m) / T in units of 1, v <= m, m finite
BQ_DEV float exponent(float v, float m, float T) {
    return T >= 1.f ? (v == -INFINITY ? v : (0.25f * v - 0.25f * m) / T * 4.f) : (v - m) / T;
}
BQ_DEV float temperature_of(const LogprobP& p, int row) { return p.temp ? p.temp[row] : 1.f; }

BQ_DEV float wave_max(float v) {
    v = fmaxf(v, dpp_f<0xB1, 0xF, true>(v));   // quad_perm [1,0,3,2]
    v = fmaxf(v, dpp_f<0x4E, 0xF, true>(v));   // quad_perm [2,3,0,1]
    v = fmaxf(v, dpp_f<0x141, 0xF, true>(v));  // row_half_mirror
    v = fmaxf(v, dpp_f<0x140, 0xF, true>(v));  // row_mirror
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
BQ_DEV int wave_min(int v) {
    for (int d = 1; d < 64; d <<= 1) v = min(v, __shfl_xor(v, d, 64));
    return v;
}

__global__ void __launch_bounds__(256) k_logprob_scan(LogprobP p) {
    constexpr int V = kSlice / 1024;  // 16-byte loads of a thread
    __shared__ float s_max[4], s_sum[4], s_dot[4];
    __shared__ uint32_t s_t[4];
    __shared__ int s_first[4], s_before[4], s_count[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, slice = blockIdx.x, row = blockIdx.y;
    const float* x = p.logits + (size_t)row * p.ld;
    auto at = [&](int k) { return slice * kSlice + (k * 256 + tid) * 4; };
    float v[V][4];
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
    const float T = temperature_of(p, row);
    const int token = p.tokens ? p.tokens[row] : -1;
    const bool given = (unsigned)token < (unsigned)p.vocab;
    const float given_v = given ? clean(x[token]) : INFINITY;

    float mine = v[0][0];
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) mine = fmaxf(mine, v[k][e]);
    const float wmax = wave_max(mine);
    if (p.top > 1) {
        // the wave's threshold: the largest 16-bit prefix of the ordered bits that `top`
        // of its lanes' maxima reach
        uint32_t cut = 0;
        const uint32_t om = ordered(mine);
#pragma unroll
        for (int bit = 31; bit >= 16; --bit) {
            const uint32_t c = cut | 1u << bit;
            if (__popcll(__ballot(om >= c)) >= p.top) cut = c;
        }
        if (lane == 0) s_t[wave] = cut;
    }
    if (lane == 0) s_max[wave] = wmax;
    __syncthreads();
    const float mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
    int first = 0x7FFFFFFF;
    if (__any(mine == mx)) {
#pragma unroll
        for (int k = V - 1; k >= 0; --k)
#pragma unroll
            for (int e = 3; e >= 0; --e)
                if (v[k][e] == mx) first = at(k) + e;
        first = wave_min(first);
    }
    int before = 0;
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) before += v[k][e] > given_v || (v[k][e] == given_v && at(k) + e < token);
    if (lane == 0) s_first[wave] = first;
    __syncthreads();
    first = min(min(s_first[0], s_first[1]), min(s_first[2], s_first[3]));

    float sum = 0.f, dot = 0.f;
    if (mx > -INFINITY && mx < INFINITY && T > 0.f) {
        const Scaled to(T);
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float y = to.y(v[k][e], mx), w = at(k) + e == first ? 0.f : __builtin_amdgcn_exp2f(y);
                sum += w;
                dot = __builtin_fmaf(w, y, dot);
            }
    }
    sum = wave_sum_dpp63(sum);
    dot = wave_sum_dpp63(dot);
    for (int d = 1; d < 64; d <<= 1) before += __shfl_xor(before, d, 64);
    if (lane == 63) {
        s_sum[wave] = sum;
        s_dot[wave] = dot;
        s_before[wave] = before;
    }
    int total = 0;
    uint32_t t = 0;
    if (p.top > 1) {
        t = max(max(s_t[0], s_t[1]), max(s_t[2], s_t[3]));
        int turn = 0;
        // tokens of the slice that satisfy f, over the workgroup
        auto count = [&](auto f) {
            int n = 0;
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < 4; ++e) n += __popcll(__ballot(at(k) + e < p.vocab && f(ordered(v[k][e]), at(k) + e)));
            turn ^= 1;
            if (lane == 0) s_count[turn][wave] = n;
            __syncthreads();
            return s_count[turn][0] + s_count[turn][1] + s_count[turn][2] + s_count[turn][3];
        };
        int last = 0x7FFFFFFF;  // of the logits that equal t, those up to this index
        total = count([&](uint32_t o, int) { return o >= t; });
        if (total > 1 << p.cap_log) {
            t = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t c = t | 1u << bit;
                if (count([&](uint32_t o, int) { return o >= c; }) >= p.top) t = c;
            }
            const int want = p.top - count([&](uint32_t o, int) { return o > t; });
            last = slice * kSlice - 1;
            for (int step = kSlice / 2; step > 0; step >>= 1)  // the most that hold fewer than wanted, and one more
                if (count([&](uint32_t o, int i) { return o == t && i <= last + step; }) < want) last += step;
            ++last;
            total = count([&](uint32_t o, int i) { return o > t || (o == t && i <= last); });
        }
        u64* cand = p.cand + (((size_t)row * p.slices + slice) << p.cap_log);
        for (int w = 0; w < wave; ++w) cand += s_count[turn][w];
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t o = ordered(v[k][e]);
                const bool in = at(k) + e < p.vocab && (o > t || (o == t && at(k) + e <= last));
                const uint64_t mask = __ballot(in);
                if (mask == 0) continue;
                if (in) cand[__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] =
                    key_of(v[k][e], at(k) + e);
                cand += __popcll(mask);
            }
    }
    __syncthreads();
    if (tid == 0) {
        SliceInfo* info = p.info + (size_t)row * p.slices + slice;
        info->best = key_of(mx, first);
        info->sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
        info->dot = (s_dot[0] + s_dot[1]) + (s_dot[2] + s_dot[3]);
        info->t = t;
        info->before = s_before[0] + s_before[1] + s_before[2] + s_before[3];
        info->count = total;
    }
}

BQ_DEV u64 larger(u64 a, u64 b) { return a > b ? a : b; }

__global__ void __launch_bounds__(256) k_logprob_join(LogprobP p) {
    __shared__ u64 s_key[kKeys], s_top[BQ_MAX_TOP], s_best[4];
    __shared__ uint32_t s_t[4];
    __shared__ float s_sum[4], s_dot[4];
    __shared__ int s_before[4], s_n;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x;
    const SliceInfo* info = p.info + (size_t)row * p.slices;
    // at most 256 slices (the entry point's limit on the vocabulary): one a thread
    SliceInfo mine = {};
    if (tid < p.slices) mine = info[tid];
    u64 best = mine.best;
    uint32_t t = mine.t;
    int before = mine.before;
    for (int d = 1; d < 64; d <<= 1) {
        best = larger(best, (u64)__shfl_xor((uint32_t)(best >> 32), d, 64) << 32 | __shfl_xor((uint32_t)best, d, 64));
        t = max(t, (uint32_t)__shfl_xor(t, d, 64));
        before += __shfl_xor(before, d, 64);
    }
    if (lane == 0) {
        s_best[wave] = best;
        s_t[wave] = t;
        s_before[wave] = before;
    }
    if (tid == 0) s_n = 0;
    __syncthreads();
    best = larger(larger(s_best[0], s_best[1]), larger(s_best[2], s_best[3]));
    t = max(max(s_t[0], s_t[1]), max(s_t[2], s_t[3]));
    const float T = temperature_of(p, row), M = value_of(best);
    // only the first token has probability: no temperature, an infinite logit, or none above -inf
    const bool sure = !(T > 0.f) || !(M > -INFINITY && M < INFINITY);
    float sum = 0.f, dot = 0.f;
    if (!sure && tid < p.slices && value_of(mine.best) > -INFINITY) {
        const Scaled to(T);
        const float y = to.y(value_of(mine.best), M), w = __builtin_amdgcn_exp2f(y), own = mine.best == best ? 0.f : 1.f;
        sum = w * (mine.sum + own);
        dot = w * (mine.dot + y * (mine.sum + own));
    }
    sum = wave_sum_dpp63(sum);
    dot = wave_sum_dpp63(dot);
    if (lane == 63) {
        s_sum[wave] = sum;
        s_dot[wave] = dot;
    }
    __syncthreads();
    sum = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
    dot = (s_dot[0] + s_dot[1]) + (s_dot[2] + s_dot[3]);
    const float log_z = log1pf(sum);
    auto log_p = [&](float v, int i) {
        if (sure) return i == index_of(best) ? 0.f : -INFINITY;
        return exponent(v, M, T) - log_z;
    };
    if (tid == 0) {
        if (p.entropy) p.entropy[row] = sure ? 0.f : log_z - 0.693147180559945309f * dot / (1.f + sum);
        if (p.tokens) {
            const int token = p.tokens[row];
            const bool given = (unsigned)token < (unsigned)p.vocab;
            if (p.logprob) p.logprob[row] = given ? log_p(clean(p.logits[(size_t)row * p.ld + token]), token) : -INFINITY;
            if (p.rank) p.rank[row] = given ? s_before[0] + s_before[1] + s_before[2] + s_before[3] : p.vocab;
        }
    }
    if (p.top == 0) return;
    int n = 1;
    if (p.top == 1) {
        if (tid == 0) s_top[0] = best;
    } else {
        // candidates not below t into s_key; where another step's might not fit, the `top`
        // largest of those found replace them
        auto cut = [&] {
            n = s_n;
            for (int i = tid; i < n; i += 256) {
                const u64 key = s_key[i];
                int rank = 0;
                for (int j = 0; j < n; ++j) rank += s_key[j] > key;
                if (rank < p.top) s_top[rank] = key;
            }
            n = min(n, p.top);
            __syncthreads();
        };
        const int slots = p.slices << p.cap_log;
        const u64* cand = p.cand + ((size_t)row * p.slices << p.cap_log);
        for (int e0 = 0; e0 < slots; e0 += kStep) {
#pragma unroll
            for (int i = 0; i < kStep / 256; ++i) {
                const int e = e0 + 256 * i + tid, s = e >> p.cap_log;
                if (e < slots && (e & ((1 << p.cap_log) - 1)) < info[s].count) {
                    const u64 key = cand[e];
                    if ((uint32_t)(key >> 32) >= t) s_key[atomicAdd(&s_n, 1)] = key;
                }
            }
            __syncthreads();
            if (s_n > kKeys - kStep && e0 + kStep < slots) {
                cut();
                for (int i = tid; i < n; i += 256) s_key[i] = s_top[i];
                if (tid == 0) s_n = n;
            }
            __syncthreads();
        }
        cut();
    }
    __syncthreads();
    for (int i = tid; i < p.top; i += 256) {
        const u64 key = i < n ? s_top[i] : 0;
        const int token = i < n ? index_of(key) : -1;
        if (p.top_tokens) p.top_tokens[(size_t)row * p.top + i] = token;
        if (p.top_logprobs) p.top_logprobs[(size_t)row * p.top + i] = i < n ? log_p(value_of(key), token) : -INFINITY;
    }
}

int slices_of(int vocab) { return (vocab + kSlice - 1) / kSlice; }
// room for a slice's candidates: about 1.5 `top` of a slice of independent logits, 3 `top`
// hardly ever
int cap_log_of(int top) {
    int n = 6;
    while (1 << n < 4 * top) ++n;
    return n;
}
}  // namespace

size_t logprob_work_bytes(int rows, int vocab, int top) {
    const size_t slices = (size_t)rows * slices_of(vocab);
    return slices * sizeof(SliceInfo) + (top > 1 ? slices << cap_log_of(top) : 0) * sizeof(u64);
}

hipError_t launch_logprobs(const bq_logprobs_args& a, hipStream_t st) {
    LogprobP p;
    p.logits = a.logits; p.ld = a.ld; p.vocab = a.vocab; p.slices = slices_of(a.vocab); p.top = a.top; p.cap_log = cap_log_of(a.top);
    p.temp = a.temperature; p.tokens = a.tokens; p.logprob = a.logprob; p.rank = a.rank; p.entropy = a.entropy;
    p.top_tokens = a.top_tokens; p.top_logprobs = a.top_logprobs;
    p.info = (SliceInfo*)a.work;
    p.cand = (u64*)(p.info + (size_t)a.rows * p.slices);
    launch_kernel(k_logprob_scan, dim3(p.slices, a.rows), dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    launch_kernel(k_logprob_join, dim3(a.rows), dim3(256), 0, st, p);
    return hipGetLastError();
}

}  // namespace bq
