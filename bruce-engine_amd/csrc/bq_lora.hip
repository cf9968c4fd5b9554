// bq_lora.hip -- low-rank adapters of many requests at once beside a projection.
//
//   y_p[r] = base_p[r] + scale[a] B_p[a] t,  t = A_p[a] x[r],  a = adapter[r]
// Two launches: k_lora_down forms t (rank values per row and part) into the
// workspace, k_lora_up adds B t.  Both are 16x16x32 bf16 MFMA with the adapter's
// rows as the A operand and 16 rows of one adapter as the B operand, so a lane holds
// one row's results, four neighbours at a time.
//
// fp32 precision on bf16 operands: the adapters and int8 codes are exact; a 32-value
// group of a q8 row is one MFMA of its codes, scaled in fp32; fp32 rows and t are the
// sum of three bf16 parts (all 24 bits), an MFMA each.
//
// Rows of one adapter are found by each workgroup itself: of up to kGather rows the
// first that has an adapter takes all that share it, from anywhere in the batch (a
// decode step's rows); of more, a workgroup takes 16 neighbours and their adapters
// one after the other (prompts: nearly always one).
#include <algorithm>

#include "bq_internal.hpp"
#include "bq_kv.hpp"

namespace bq {

namespace {
constexpr int kGather = 256;
constexpr int kRankTiles = 4;  // 16-rank tiles of a workgroup of k_lora_down at most
constexpr int kUpTiles = 4;    // 16-output tiles of a wave of k_lora_up

enum XKind { kXQ8, kXF32, kXBf16 };

struct LoraP {
    const void* x;
    const float* xd;
    int64_t ldx;
    const int32_t* adapter;
    const float* scale;
    const uint16_t* a[kMaxParts];
    const uint16_t* b[kMaxParts];
    const float* base[kMaxParts];
    float* y[kMaxParts];
    int64_t ldbase[kMaxParts], ldy[kMaxParts];
    int N[kMaxParts], chunk0[kMaxParts];  // first output chunk of a part
    int n_parts, rows, K, rank, n_adapters;
    float* t;  // [rows][n_parts][rank]
};

BQ_DEV f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// a row's adapter, -1: none
BQ_DEV int adapter_of(const LoraP& p, int r) {
    const int a = p.adapter[r];
    return (unsigned)a < (unsigned)p.n_adapters ? a : -1;
}

// Calls f(adapter, rows, n) for this workgroup's rows, n <= 16 of one adapter at a
// time (rows in LDS).  All of the workgroup's lanes take part; f may hold barriers.
template <typename F>
BQ_DEV void each_adapter(const LoraP& p, int* s_rows, int* s_n, F f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (p.rows <= kGather) {
        const int me = blockIdx.x, a = adapter_of(p, me);
        if (wave == 0) {
            int n = 0;
            for (int r0 = 0; r0 < p.rows; r0 += 64) {
                const int r = r0 + lane;
                const uint64_t same = __ballot(r < p.rows && adapter_of(p, min(r, p.rows - 1)) == a);
                if (same >> lane & 1) s_rows[n + __builtin_popcountll(same & ((1ull << lane) - 1))] = r;
                n += __builtin_popcountll(same);
            }
            if (lane == 0) *s_n = n;
        }
        __syncthreads();
        if (s_rows[0] != me) return;
        const int n = *s_n;
        for (int i = 0; i < n; i += 16) f(a, s_rows + i, min(16, n - i));
    } else {
        const int r0 = blockIdx.x * 16, n = min(16, p.rows - r0), a = adapter_of(p, r0 + min(lane & 15, n - 1));
        uint32_t left = (1u << n) - 1;
        while (left) {
            const int one = __builtin_amdgcn_readlane(a, __builtin_ctz(left));
            const uint32_t same = (uint32_t)__ballot(a == one) & left;
            left &= ~same;
            if (wave == 0 && lane < 16 && (same >> lane & 1)) s_rows[__builtin_popcount(same & ((1u << lane) - 1))] = r0 + lane;
            __syncthreads();
            f(one, s_rows, __builtin_popcount(same));
            __syncthreads();
        }
    }
}

// the three bf16 parts of 8 floats, largest first: each takes the leading 8 bits of what is left
BQ_DEV void parts_of(f32x4 lo, f32x4 hi, bf16x8 (&out)[3]) {
    float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            w[e] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x[2 * e + 1]), __builtin_bit_cast(uint32_t, x[2 * e]), 0x07060302u);
            x[2 * e] -= as_float(w[e] << 16);
            x[2 * e + 1] -= as_float(w[e] & 0xFFFF0000u);
        }
        out[n] = __builtin_bit_cast(bf16x8, w);
    }
}
BQ_DEV u32x2 codes_bf16(uint32_t w) {
    const float a = (float)(int8_t)w, b = (float)(int8_t)(w >> 8), c = (float)(int8_t)(w >> 16), d = (float)((int32_t)w >> 24);
    auto hi2 = [](float x, float y) {  // the high halves: small integers are exact in bf16
        return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, y), __builtin_bit_cast(uint32_t, x), 0x07060302u);
    };
    return u32x2{hi2(a, b), hi2(c, d)};
}

// t: a workgroup has up to 16 TILES ranks of one part; its waves share K.  (The number of
// tiles is fixed when it is compiled: with a branch between an MFMA and the first use of
// its result the compiler has left out the wait that the result needs.)
template <int X, int TILES>
__global__ void __launch_bounds__(256) k_lora_down(LoraP p) {
    __shared__ int s_rows[kGather], s_n;
    __shared__ __attribute__((aligned(16))) float s_t[4][16][16 * TILES + 4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
    const int chunks = (p.rank + 16 * TILES - 1) / (16 * TILES), part = blockIdx.y / chunks, j0 = blockIdx.y % chunks * 16 * TILES;
    const int nj = min(16 * TILES, p.rank - j0);
    const int steps = p.K / 32;
    each_adapter(p, s_rows, &s_n, [&](int a, const int* rows, int n) {
        if (a < 0) return;
        const int64_t row = rows[min(c, n - 1)];
        const uint16_t* A[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i)  // ranks past the last read it again; they are not stored
            A[i] = p.a[part] + ((int64_t)a * p.rank + min(j0 + 16 * i + c, p.rank - 1)) * p.K + 8 * g;
        f32x4 t[TILES];
#pragma unroll
        for (int i = 0; i < TILES; ++i) t[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s = wave; s < steps; s += 4) {
            const int k = 32 * s;
            bf16x8 xp[3];
            float d = 1.f;
            if constexpr (X == kXQ8) {
                const u32x2 w = *(const u32x2*)((const char*)p.x + row * p.K + k + 8 * g);
                const u32x2 lo = codes_bf16(w[0]), hi = codes_bf16(w[1]);
                xp[0] = __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
                d = p.xd[row * steps + s];
            } else if constexpr (X == kXF32) {
                const float* x = (const float*)p.x + row * p.ldx + k + 8 * g;
                parts_of(*(const f32x4*)x, *(const f32x4*)(x + 4), xp);
            } else {
                xp[0] = __builtin_bit_cast(bf16x8, *(const u32x4*)((const uint16_t*)p.x + row * p.ldx + k + 8 * g));
            }
#pragma unroll
            for (int i = 0; i < TILES; ++i) {
                const bf16x8 w = __builtin_bit_cast(bf16x8, *(const u32x4*)(A[i] + k));
                if constexpr (X == kXQ8) {
                    t[i] += mfma16(w, xp[0], f32x4{0.f, 0.f, 0.f, 0.f}) * d;
                } else {
#pragma unroll
                    for (int q = X == kXF32 ? 2 : 0; q >= 0; --q) t[i] = mfma16(w, xp[q], t[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < TILES; ++i) *(f32x4*)&s_t[wave][c][16 * i + 4 * g] = t[i];
        __syncthreads();
        const float scale = p.scale ? p.scale[a] : 1.f;
        for (int e = tid; e < n * nj; e += 256) {
            const int r = e / nj, j = e % nj;
            const float v = (s_t[0][r][j] + s_t[1][r][j]) + (s_t[2][r][j] + s_t[3][r][j]);
            p.t[((int64_t)rows[r] * p.n_parts + part) * p.rank + j0 + j] = v * scale;
        }
        __syncthreads();
    });
}

// y: a wave has kUpTiles tiles of 16 outputs of one part
__global__ void __launch_bounds__(256) k_lora_up(LoraP p) {
    __shared__ int s_rows[kGather], s_n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    int part = 0;
    while (part + 1 < p.n_parts && (int)blockIdx.y >= p.chunk0[part + 1]) ++part;
    const int n0 = (((int)blockIdx.y - p.chunk0[part]) * 4 + wave) * 16 * kUpTiles, N = p.N[part];
    const float* base = p.base[part];
    float* y = p.y[part];
    each_adapter(p, s_rows, &s_n, [&](int a, const int* rows, int n) {
        if (a < 0 && base == y) return;
        const bool live = c < n;
        const int64_t row = rows[min(c, n - 1)];
        f32x4 acc[kUpTiles];
#pragma unroll
        for (int i = 0; i < kUpTiles; ++i) {
            acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int o = n0 + 16 * i + 4 * g;
            if (base && live && o < N) acc[i] = *(const f32x4*)(base + row * p.ldbase[part] + o);
        }
        if (a >= 0) {
            const float* t = p.t + (row * p.n_parts + part) * p.rank;
            const uint16_t* B = p.b[part] + (int64_t)a * N * p.rank;
            for (int k = 8 * g; k < (p.rank + 31 & ~31); k += 32) {
                const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                bf16x8 tp[3];
                parts_of(k < p.rank ? *(const f32x4*)(t + k) : zero, k < p.rank ? *(const f32x4*)(t + k + 4) : zero, tp);
#pragma unroll
                for (int i = 0; i < kUpTiles; ++i) {
                    const int o = n0 + 16 * i + c;
                    const u32x4 w = k < p.rank && o < N ? *(const u32x4*)(B + (int64_t)o * p.rank + k) : u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int q = 2; q >= 0; --q) acc[i] = mfma16(__builtin_bit_cast(bf16x8, w), tp[q], acc[i]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kUpTiles; ++i) {
            const int o = n0 + 16 * i + 4 * g;
            if (live && o < N) *(f32x4*)(y + row * p.ldy[part] + o) = acc[i];
        }
    });
}
template <int X>
void launch_down(const LoraP& p, int tiles, dim3 grid, hipStream_t st) {
    switch (tiles) {
        case 1: launch_kernel((k_lora_down<X, 1>), grid, dim3(256), 0, st, p); break;
        case 2: launch_kernel((k_lora_down<X, 2>), grid, dim3(256), 0, st, p); break;
        case 3: launch_kernel((k_lora_down<X, 3>), grid, dim3(256), 0, st, p); break;
        default: launch_kernel((k_lora_down<X, 4>), grid, dim3(256), 0, st, p);
    }
}
}  // namespace

size_t lora_work_bytes(int rows, int rank, int n_parts) { return (size_t)rows * n_parts * rank * sizeof(float); }

hipError_t launch_lora(const bq_lora_args& a, hipStream_t st) {
    LoraP p;
    p.x = a.x; p.xd = a.xd; p.ldx = a.ldx; p.adapter = a.adapter; p.scale = a.scale;
    p.n_parts = a.n_parts; p.rows = a.rows; p.K = a.K; p.rank = a.rank; p.n_adapters = a.n_adapters; p.t = (float*)a.work;
    int chunks = 0;
    for (int i = 0; i < a.n_parts; ++i) {
        const bq_lora_part& q = a.parts[i];
        p.a[i] = q.a; p.b[i] = q.b; p.base[i] = q.base; p.y[i] = q.y; p.ldbase[i] = q.ldbase; p.ldy[i] = q.ldy; p.N[i] = q.N;
        p.chunk0[i] = chunks;
        chunks += (q.N + 64 * kUpTiles - 1) / (64 * kUpTiles);
    }
    const uint32_t groups = a.rows <= kGather ? a.rows : (a.rows + 15) / 16;
    const int tiles = std::min((a.rank + 15) / 16, kRankTiles);
    const dim3 down(groups, a.n_parts * ((a.rank + 16 * tiles - 1) / (16 * tiles)));
    switch (a.x_type) {
        case BQ_TYPE_Q8_0: launch_down<kXQ8>(p, tiles, down, st); break;
        case BQ_TYPE_F32: launch_down<kXF32>(p, tiles, down, st); break;
        default: launch_down<kXBf16>(p, tiles, down, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    launch_kernel(k_lora_up, dim3(groups, chunks), dim3(256), 0, st, p);
    return hipGetLastError();
}

}  // namespace bq
