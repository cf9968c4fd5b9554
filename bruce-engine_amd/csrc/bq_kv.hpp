// bq_kv.hpp -- device view of the paged key-value cache (layout: include/bq.h)
// and the bf16 helpers of the kernels that read and write it.
#pragma once
#include "bq_device.hpp"

namespace bq {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

enum KvType { kKvBf16 = 0, kKvQ8 = 1 };

struct KvView {
    char* pages;
    const int32_t* table;
    int64_t page_bytes;
    int head_bytes;  // one head's keys and values in a page
    int heads, D, P, plog;
    int n_pages, n_seq, max_pages;
};

// page of a token, -1 if there is none (an unmapped entry, a sequence or a
// token outside the table)
BQ_DEV int kv_page(const KvView& kv, int seq, int tok) {
    if ((unsigned)seq >= (unsigned)kv.n_seq || tok < 0 || (tok >> kv.plog) >= kv.max_pages) return -1;
    const int id = kv.table[(size_t)seq * kv.max_pages + (tok >> kv.plog)];
    return (unsigned)id < (unsigned)kv.n_pages ? id : -1;
}

// bytes from a head's start in a page (P tokens of D values) to
// bf16: the 16-byte unit of dims 8c..8c+7 of token t / of tokens 8t..8t+7 of dim d
BQ_DEV int kv_k_unit(int P, int c, int t) { return (c * P + t) * 16; }
BQ_DEV int kv_v_unit(int P, int D, int t8, int d) { return P * D * 2 + (t8 * D + d) * 16; }
// q8: the unit of K codes (c, g) of token t, of V codes (t8, c, m), and the scales of dims 32c..32c+31
BQ_DEV int kv_kq_unit(int P, int c, int g, int t) { return ((c * 4 + g) * P + t) * 16; }
BQ_DEV int kv_vq_unit(int P, int D, int t8, int c, int m) { return P * D + ((t8 * (D / 32) + c) * 16 + m) * 16; }
BQ_DEV int kv_ks_off(int P, int D, int c, int t) { return 2 * P * D + (c * P + t) * 2; }
BQ_DEV int kv_vs_off(int P, int D, int c, int t) { return 2 * P * D + (D / 32 * P + c * P + t) * 2; }

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
BQ_DEV float pow2(int e) { return as_float((uint32_t)(e + 127) << 23); }                           // |e| <= 126
BQ_DEV int ilogb2(float x) { return (int)(__builtin_bit_cast(uint32_t, x) >> 23 & 0xFF) - 127; }  // of a normal x

// four int8 codes -> fp16: a byte c ^ 0x80 under the exponent of 1024 is
// 1024 + 128 + c, exactly
BQ_DEV void codes_f16(uint32_t w, f16x2& lo, f16x2& hi) {
    w ^= 0x80808080u;
    const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    lo = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
    hi = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
}

BQ_DEV uint16_t f2bf(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
BQ_DEV float bf2f(uint16_t b) { return as_float((uint32_t)b << 16); }
BQ_DEV uint32_t f2bf2(float a, float b) {
    const bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
}

}  // namespace bq
