// A cache in blocks of tokens: keys and values into it and back.
//
// A block and kv head holds e4m3 codes of x * 2^-e with one e for its keys and one for its values, the least for which the
// largest magnitude fits 448.  With a power of two the scaling is exact, so a value is rounded once, to the nearest of
// what e4m3 holds (half a step: 2^-4 of the value), and where a later token raises e the codes before it move to the
// new scale without loss, those aside that become subnormal and round once more.  No border depends on the order of an
// f32 sum or on a division.
//
// Store: memory-bound.  A workgroup takes one run of tokens inside one block (the first of the run's tokens finds that it is the
// first from the slots alone), one kv head, keys or values: what shares an e is then one workgroup's, and its largest
// magnitude is known before the first code is written, with the values held in registers.
#include "common.hpp"
#include "lanes.hpp"
#include "paged_device.hpp"

namespace saetta {
namespace {

constexpr int STORE_THREADS = 256;

struct StoreArgs {
    saetta_strided_rows x[2];  // keys, values
    const int32_t *slots;
    uint8_t *codes[2], *scales[2];
    uint32_t blocks, block_tokens, kv_heads, tokens;
};

// Values of one unit of 16 tokens that a thread holds.  Keys: 16 dims of one token, a piece of 16 bytes.  Values: four dims
// of four tokens, a dword of each of four pieces.
struct KeyPlace {
    static constexpr bool KEYS = true;
    uint32_t token, dim;
    __device__ __forceinline__ KeyPlace(uint32_t tid) : token(tid >> 4), dim((tid & 15) * 16) {}
    __device__ __forceinline__ uint32_t byte() const { return dim / 64 * 1024 + (dim / 16 % 4 * 16 + token) * 16; }
};
struct ValuePlace {
    static constexpr bool KEYS = false;
    uint32_t token, dim;  // the first of four
    // (lanes: dims of 64 side by side, 4 at a time, then the four 64s: what a token has is read whole)
    __device__ __forceinline__ ValuePlace(uint32_t tid) : token((tid >> 6) * 4), dim((tid & 63) * 4) {}
    __device__ __forceinline__ uint32_t byte() const { return dim / 64 * 1024 + (token / 4 * 16 + dim % 16) * 16 + dim / 16 % 4 * 4; }
};

template <int TYPE, int UNITS, class Place>
__device__ __forceinline__ void store_run(const StoreArgs &a, int which, uint32_t token, uint32_t head, uint32_t block, uint32_t offset, uint32_t count) {
    typedef typename Row<TYPE>::value V;
    const uint32_t tid = threadIdx.x;
    const Place place(tid);
    const saetta_strided_rows &rows = a.x[which];
    // the run's token 0 sits at `offset`; token t of the block is row t - offset of the run
    const V *x = static_cast<const V *>(rows.data) + uint64_t(token) * rows.token_stride + head * rows.head_stride + place.dim;
    float held[UNITS][16];
    float top = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        if constexpr (Place::KEYS) {
            const uint32_t t = u * UNIT_TOKENS + place.token;
            if (t >= offset && t < offset + count) load_values<TYPE, 16>(x + uint64_t(t - offset) * rows.token_stride, held[u]);
            else {
#pragma unroll
                for (int i = 0; i < 16; i++) held[u][i] = 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t t = u * UNIT_TOKENS + place.token + i;
                float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                if (t >= offset && t < offset + count) load_values<TYPE, 4>(x + uint64_t(t - offset) * rows.token_stride, v);
#pragma unroll
                for (int d = 0; d < 4; d++) held[u][4 * d + i] = v[d];
            }
        }
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const float m = fabsf(held[u][i]);
            top = m < __builtin_inff() ? fmaxf(top, m) : top;
        }
    }
    top = group_reduce<64>(top, MaxOp());
    __shared__ float tops[STORE_THREADS / 64];
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < STORE_THREADS / 64; w++) top = fmaxf(top, tops[w]);

    const size_t at = size_t(block) * a.kv_heads + head;
    uint8_t *scale = a.scales[which] + at;
    const int before = int(*scale) - 127;
    int e = scale_exponent(top);
    if (offset > 0) e = max(e, min(max(before, LOWEST_EXPONENT), HIGHEST_EXPONENT));
    const bool raised = offset > 0 && e != before;
    const float down = power_of_two(-e), moved = power_of_two(max(before - e, -126));
    uint8_t *codes = a.codes[which] + at * (size_t(a.block_tokens) * SAETTA_HEAD_DIM);
#pragma unroll
    for (int u = 0; u < UNITS; u++) {
        const uint32_t first = u * UNIT_TOKENS;
        // nothing of the unit is new, nor to be moved to another scale
        if (first >= offset + count || (first + UNIT_TOKENS <= offset && !raised)) continue;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = to_codes(held[u][4 * i] * down, held[u][4 * i + 1] * down, held[u][4 * i + 2] * down, held[u][4 * i + 3] * down);
        uint8_t *to = codes + u * UNIT_BYTES + place.byte();
        auto rescaled = [&](uint32_t old) {
            float v[4];
            of_codes(old, v);
            return to_codes(v[0] * moved, v[1] * moved, v[2] * moved, v[3] * moved);
        };
        if constexpr (Place::KEYS) {
            const uint32_t t = first + place.token;
            if (t >= offset + count) continue;
            uint4 *piece = reinterpret_cast<uint4 *>(to);
            if (t >= offset) {
                *piece = uint4{w[0], w[1], w[2], w[3]};
            } else if (raised) {
                const uint4 old = *piece;
                *piece = uint4{rescaled(old.x), rescaled(old.y), rescaled(old.z), rescaled(old.w)};
            }
        } else {
            const uint32_t t = first + place.token;
            if (t >= offset + count || (t + 4 <= offset && !raised)) continue;
            const bool whole = t >= offset && t + 4 <= offset + count;
            uint32_t fresh = 0, earlier = 0;  // bytes of tokens that are new; of tokens before them
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (t + i < offset) earlier |= 0xffu << (8 * i);
                else if (t + i < offset + count) fresh |= 0xffu << (8 * i);
            }
#pragma unroll
            for (int d = 0; d < 4; d++) {
                uint32_t *p = reinterpret_cast<uint32_t *>(to + d * 16), value = w[d];
                if (!whole) {
                    const uint32_t old = *p, kept = raised ? rescaled(old) : old;
                    value = (value & fresh) | (kept & earlier) | (old & ~(fresh | earlier));
                }
                *p = value;
            }
        }
    }
    if (tid == 0) *scale = uint8_t(e + 127);
}

template <int TYPE, int UNITS>
__global__ __launch_bounds__(STORE_THREADS) void paged_store_kernel(StoreArgs a) {
    const uint32_t token = blockIdx.x, head = blockIdx.y >> 1;
    const int which = blockIdx.y & 1;
    const uint32_t slot = uint32_t(a.slots[token]), bt = UNITS * UNIT_TOKENS;
    const uint32_t block = slot / bt, offset = slot % bt;
    if (block >= a.blocks) return;  // (-1 among them)
    // the run's first token: what is before it in the call is in another block, or not the slot before
    if (offset > 0 && token > 0 && uint32_t(a.slots[token - 1]) == slot - 1) return;
    __shared__ uint32_t found;
    // the tokens that follow it in the block, slot by slot: one wave looks at up to 64 at a time
    if (threadIdx.x < 64) {
        uint32_t count = 1;
        for (uint32_t i0 = 1; i0 < bt - offset; i0 += 64) {
            const uint32_t i = i0 + threadIdx.x;
            const bool follows = i < bt - offset && uint64_t(token) + i < a.tokens && uint32_t(a.slots[token + i]) == slot + i;
            const uint64_t all = __ballot(follows);
            const uint32_t n = all == ~0ull ? 64 : uint32_t(__builtin_ctzll(~all));
            count += n;
            if (n < 64) break;
        }
        if (threadIdx.x == 0) found = count;
    }
    __syncthreads();
    const uint32_t count = found;
    if (which == 0) store_run<TYPE, UNITS, KeyPlace>(a, 0, token, head, block, offset, count);
    else store_run<TYPE, UNITS, ValuePlace>(a, 1, token, head, block, offset, count);
}

struct GatherArgs {
    const uint8_t *codes[2], *scales[2];
    const int32_t *slots;
    void *out[2];
    uint32_t blocks, block_tokens, kv_heads, tokens;
};

// A workgroup takes 16 slots of one kv head, keys or values, a thread 16 dims of a slot.
template <int TYPE>
__global__ __launch_bounds__(256) void paged_gather_kernel(GatherArgs a) {
    typedef typename Row<TYPE>::value V;
    const uint32_t tid = threadIdx.x, head = blockIdx.y >> 1, which = blockIdx.y & 1;
    const uint64_t row = uint64_t(blockIdx.x) * 16 + (tid >> 4);
    if (row >= a.tokens || a.out[which] == nullptr) return;
    const uint32_t slot = uint32_t(a.slots[row]), block = slot / a.block_tokens;
    if (block >= a.blocks) return;
    const size_t at = size_t(block) * a.kv_heads + head;
    const uint8_t *unit = a.codes[which] + at * (size_t(a.block_tokens) * SAETTA_HEAD_DIM) + slot % a.block_tokens / UNIT_TOKENS * UNIT_BYTES;
    const float scale = power_of_two(int(a.scales[which][at]) - 127);
    const uint32_t t = slot % UNIT_TOKENS, piece = tid & 15;  // dims 16 piece ..
    float x[16];
    if (which == 0) {
        const uint4 w = *reinterpret_cast<const uint4 *>(unit + (piece >> 2) * 1024 + ((piece & 3) * 16 + t) * 16);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v[4];
            of_codes(ws[i], v);
#pragma unroll
            for (int j = 0; j < 4; j++) x[4 * i + j] = v[j] * scale;
        }
    } else {
        const uint8_t *p = unit + (piece >> 2) * 1024 + (t >> 2) * 256 + (piece & 3) * 4 + (t & 3);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const uint32_t w = uint32_t(p[i * 16]) | uint32_t(p[i * 16 + 16]) << 8 | uint32_t(p[i * 16 + 32]) << 16 | uint32_t(p[i * 16 + 48]) << 24;
            float v[4];
            of_codes(w, v);
#pragma unroll
            for (int j = 0; j < 4; j++) x[i + j] = v[j] * scale;
        }
    }
    store_values<TYPE, 16>(static_cast<V *>(a.out[which]) + (row * a.kv_heads + head) * SAETTA_HEAD_DIM + piece * 16, x);
}

template <int TYPE>
void launch_store(hipStream_t stream, const StoreArgs &a) {
    const dim3 grid(a.tokens, a.kv_heads * 2);
    switch (a.block_tokens) {
        case 16: return launch(paged_store_kernel<TYPE, 1>, grid, dim3(STORE_THREADS), 0, stream, a);
        case 32: return launch(paged_store_kernel<TYPE, 2>, grid, dim3(STORE_THREADS), 0, stream, a);
        case 64: return launch(paged_store_kernel<TYPE, 4>, grid, dim3(STORE_THREADS), 0, stream, a);
        default: return launch(paged_store_kernel<TYPE, 8>, grid, dim3(STORE_THREADS), 0, stream, a);
    }
}

}  // namespace

int setup_paged_cache() { return load_kernel(reinterpret_cast<const void *>(paged_gather_kernel<SAETTA_F16>)); }

}  // namespace saetta

using namespace saetta;

extern "C" int saetta_paged_store(saetta_stream_t stream, int type, saetta_strided_rows keys, saetta_strided_rows values,
                                  const int32_t *slots, saetta_paged_cache cache, uint32_t tokens) {
    SAETTA_REQUIRE(type == SAETTA_F32 || type == SAETTA_F16 || type == SAETTA_BF16, SAETTA_E_BITS, "paged_store: type %d (f32, f16 or bf16)", type);
    SAETTA_REQUIRE(keys.data && values.data && slots, SAETTA_E_NULL, "paged_store: null buffer");
    if (int rc = check_cache(cache, "paged_store")) return rc;
    SAETTA_REQUIRE(aligned(slots, 4) && rows_aligned(keys, type) && rows_aligned(values, type), SAETTA_E_ALIGN,
                   "paged_store: keys and values must be 16-byte aligned, with strides of multiples of 16 bytes");
    if (int rc = ensure_device()) return rc;
    if (tokens == 0) return SAETTA_OK;
    const StoreArgs a = {{keys, values}, slots, {cache.keys, cache.values}, {cache.key_scales, cache.value_scales},
                         cache.blocks, cache.block_tokens, cache.kv_heads, tokens};
    if (type == SAETTA_F32) launch_store<SAETTA_F32>(as_stream(stream), a);
    else if (type == SAETTA_F16) launch_store<SAETTA_F16>(as_stream(stream), a);
    else launch_store<SAETTA_BF16>(as_stream(stream), a);
    return launch_status("paged_store");
}

extern "C" int saetta_paged_gather(saetta_stream_t stream, int type, saetta_paged_cache cache, const int32_t *slots, void *keys,
                                   void *values, uint32_t tokens) {
    SAETTA_REQUIRE(type == SAETTA_F32 || type == SAETTA_F16 || type == SAETTA_BF16, SAETTA_E_BITS, "paged_gather: type %d (f32, f16 or bf16)", type);
    SAETTA_REQUIRE(slots, SAETTA_E_NULL, "paged_gather: null slots");
    if (int rc = check_cache(cache, "paged_gather")) return rc;
    SAETTA_REQUIRE(aligned(slots, 4) && aligned(keys, 16) && aligned(values, 16), SAETTA_E_ALIGN, "paged_gather: keys and values must be 16-byte aligned");
    if (int rc = ensure_device()) return rc;
    if (tokens == 0 || (!keys && !values)) return SAETTA_OK;
    const GatherArgs a = {{cache.keys, cache.values}, {cache.key_scales, cache.value_scales}, slots, {keys, values},
                          cache.blocks, cache.block_tokens, cache.kv_heads, tokens};
    const dim3 grid((tokens + 15) / 16, cache.kv_heads * 2);
    if (type == SAETTA_F32) launch(paged_gather_kernel<SAETTA_F32>, grid, dim3(256), 0, as_stream(stream), a);
    else if (type == SAETTA_F16) launch(paged_gather_kernel<SAETTA_F16>, grid, dim3(256), 0, as_stream(stream), a);
    else launch(paged_gather_kernel<SAETTA_BF16>, grid, dim3(256), 0, as_stream(stream), a);
    return launch_status("paged_gather");
}
