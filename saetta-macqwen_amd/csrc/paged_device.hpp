// What the kernels over a cache in blocks share: where a code lies, what it stands for, rows of three types.
#pragma once
#include "common.hpp"

namespace saetta {

constexpr uint32_t UNIT_TOKENS = 16, UNIT_BYTES = UNIT_TOKENS * SAETTA_HEAD_DIM;
constexpr int LOWEST_EXPONENT = -40, HIGHEST_EXPONENT = 60;

inline bool block_tokens_ok(uint32_t n) { return n == 16 || n == 32 || n == 64 || n == 128; }
inline uint32_t type_bytes(int type) { return type == SAETTA_F32 ? 4 : 2; }
inline bool rows_aligned(const saetta_strided_rows &r, int type) {
    const uint64_t values = 16 / type_bytes(type);
    return aligned(r.data, 16) && r.token_stride % values == 0 && r.head_stride % values == 0;
}
// Checks that the entry points have in common; 0 or a code.
inline int check_cache(const saetta_paged_cache &c, const char *what) {
    SAETTA_REQUIRE(c.keys && c.values && c.key_scales && c.value_scales, SAETTA_E_NULL, "%s: null cache buffer", what);
    SAETTA_REQUIRE(aligned(c.keys, 16) && aligned(c.values, 16), SAETTA_E_ALIGN, "%s: keys and values must be 16-byte aligned", what);
    SAETTA_REQUIRE(block_tokens_ok(c.block_tokens), SAETTA_E_SHAPE, "%s: blocks of %u tokens (16, 32, 64 or 128)", what, c.block_tokens);
    SAETTA_REQUIRE(c.kv_heads > 0 && c.kv_heads <= 65535 / 2, SAETTA_E_SHAPE, "%s: %u kv heads", what, c.kv_heads);
    SAETTA_REQUIRE(c.blocks > 0 && uint64_t(c.blocks) * c.block_tokens < (1ull << 31), SAETTA_E_SHAPE,
                   "%s: %u blocks of %u tokens (fewer than 2^31 tokens)", what, c.blocks, c.block_tokens);
    SAETTA_REQUIRE(uint64_t(c.blocks) * c.kv_heads < (1ull << 32), SAETTA_E_SHAPE, "%s: %u blocks of %u kv heads (fewer than 2^32 in all)", what, c.blocks, c.kv_heads);
    return SAETTA_OK;
}

// The last of `starts` (rising, starts[0] <= x) that is no more than x, for N numbers at once: as many looks for each, none waiting for another's.
template <int N>
__device__ __forceinline__ void last_at_most(const uint32_t *starts, uint32_t n, const uint32_t (&x)[N], uint32_t (&low)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) low[i] = 0;
    while (n > 1) {
        const uint32_t half = n / 2;
        n -= half;  // (of an odd n the lower part keeps a place that has been looked at)
#pragma unroll
        for (int i = 0; i < N; i++) low[i] += starts[low[i] + half] <= x[i] ? half : 0;
    }
}
__device__ __forceinline__ uint32_t last_at_most(const uint32_t *starts, uint32_t n, uint32_t x) {
    const uint32_t one[1] = {x};
    uint32_t low[1];
    last_at_most(starts, n, one, low);
    return low[0];
}

typedef float floatx2 __attribute__((ext_vector_type(2)));

// 2^e as it is, for e in -126..127
__device__ __forceinline__ float power_of_two(int e) { return __builtin_bit_cast(float, uint32_t(e + 127) << 23); }

// The least e of the range with amax <= 448 * 2^e: 448 is 1.75 * 2^8, so a mantissa past 1.75 carries into the exponent.
__device__ __forceinline__ int scale_exponent(float amax) {
    const int e = int((__builtin_bit_cast(uint32_t, amax) + 0x1fffffu) >> 23) - (127 + 8);
    return min(max(e, LOWEST_EXPONENT), HIGHEST_EXPONENT);
}

// Four codes of four values of magnitudes up to 448, to nearest even; what is larger or no number becomes NaN (0x7f).
__device__ __forceinline__ uint32_t to_codes(float a, float b, float c, float d) {
    auto held = [](float x) { return fabsf(x) <= 448.0f ? x : __builtin_nanf(""); };
    const int low = __builtin_amdgcn_cvt_pk_fp8_f32(held(a), held(b), 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(held(c), held(d), low, true));
}
// ... and back
__device__ __forceinline__ void of_codes(uint32_t w, float (&x)[4]) {
    const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

template <int TYPE>
struct Row;
template <>
struct Row<SAETTA_F32> {
    typedef float value;
    static __device__ __forceinline__ float load(float x) { return x; }
    static __device__ __forceinline__ float store(float x) { return x; }
};
template <>
struct Row<SAETTA_F16> {
    typedef _Float16 value;
    static __device__ __forceinline__ float load(_Float16 x) { return float(x); }
    static __device__ __forceinline__ _Float16 store(float x) { return _Float16(x); }
};
template <>
struct Row<SAETTA_BF16> {
    typedef __bf16 value;
    static __device__ __forceinline__ float load(__bf16 x) { return float(x); }
    static __device__ __forceinline__ __bf16 store(float x) { return __bf16(x); }
};

// N values that lie side by side, 4 N or 2 N bytes aligned up to 16
template <int TYPE, int N>
__device__ __forceinline__ void load_values(const typename Row<TYPE>::value *p, float (&x)[N]) {
    typedef typename Row<TYPE>::value V;
    constexpr int PER = N * sizeof(V) < 16 ? N : 16 / sizeof(V);
    typedef V vec __attribute__((ext_vector_type(PER)));
#pragma unroll
    for (int i = 0; i < N; i += PER) {
        const vec v = *reinterpret_cast<const vec *>(p + i);
#pragma unroll
        for (int j = 0; j < PER; j++) x[i + j] = Row<TYPE>::load(v[j]);
    }
}
template <int TYPE, int N, bool PASSING = false>  // PASSING: by the caches
__device__ __forceinline__ void store_values(typename Row<TYPE>::value *p, const float (&x)[N]) {
    typedef typename Row<TYPE>::value V;
    constexpr int PER = N * sizeof(V) < 16 ? N : 16 / sizeof(V);
    typedef V vec __attribute__((ext_vector_type(PER)));
#pragma unroll
    for (int i = 0; i < N; i += PER) {
        vec v;
#pragma unroll
        for (int j = 0; j < PER; j++) v[j] = Row<TYPE>::store(x[i + j]);
        if constexpr (PASSING) __builtin_nontemporal_store(v, reinterpret_cast<vec *>(p + i));
        else *reinterpret_cast<vec *>(p + i) = v;
    }
}

}  // namespace saetta
