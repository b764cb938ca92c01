// A cache in blocks of tokens: keys and values into it and back.
//
// A block and kv head holds e4m3 codes of x * 2^-e with one e for its keys and one for its values, the least for which the
// largest magnitude fits 448.  With a power of two the scaling is exact, so a value is rounded once, to the nearest of
// what e4m3 holds (half a step: 2^-4 of the value), and where a later token raises e the codes before it move to the
// new scale without loss, those aside that become subnormal and round once more.  No border depends on the order of an
// f32 sum or on a division.
//
// Store: memory-bound.  What shares an e is one workgroup's: a run of tokens inside one block (the first of the run's tokens finds that it is the first
// from the slots alone), one kv head, keys or values; its largest magnitude is known before the first code is written, with the values held in
// registers.  A wave has four tokens of a unit, a lane four dims of each: a load is a token's row, and what a wave stores of four tokens fills lines of 64
// bytes.  A run of up to four tokens is one wave's, so that a step's tokens and drafts are stored at once.  Measured, 2 kv heads: 9700 tokens of five
// prompts, f32, blocks of 16, 13 us, 3.8 TB/s of what is read and written (a large copy: 4.9; with whole tokens to a wave, whose stores fill no lines, 22.8);
// 16384 tokens in 16 bits, blocks of 16, 32, 64 and 128, 17, 18, 20 and 48 us: a long run's loads, barrier and stores follow each other, and runs of 128 tokens
// begin in every other workgroup, so that half of the XCDs have none; 100 prompts of 90 tokens 14, 24, 22 and 33 us, by what the workgroups with several runs take; 64 single
// tokens 4.8 us, the chain of slot, row, maximum and codes, and no more in a step that has room for 4096.
#include "common.hpp"
#include "lanes.hpp"
#include "paged_device.hpp"

namespace saetta {
namespace {

// Waves of a workgroup of the store: four to a unit of tokens, of up to two units at once.
constexpr uint32_t store_waves(int units) { return 4 * (units < 2 ? units : 2); }
// A run of up to so many tokens is a wave's, so that a step of single tokens, or drafts, is stored at once.
constexpr uint32_t SHORT_RUN = 4;
// Tokens of a block, a lane a token.
constexpr uint32_t lane_tokens(int units) { return units < 4 ? units * UNIT_TOKENS : 64; }
// Workgroups (of all kv heads and sides) that look for runs, unless a block's tokens would be fewer than each looks at.
constexpr uint32_t STORE_GROUPS = 512;

// The most tokens of a call: 2^32 threads are one more than a launch has, and a workgroup of the store has 512 for 32 tokens, or 256 for 16, at most.
constexpr uint32_t MOST_TOKENS = (1u << 28) - 32;

struct StoreArgs {
    saetta_strided_rows x[2];  // keys, values
    const int32_t *slots;
    uint8_t *codes[2], *scales[2];
    uint32_t blocks, block_tokens, kv_heads, tokens;
};

// Where the four dims (from `dim` on) of token t, of keys, or dim `dim` of the four tokens from t on, of values, lie in a unit: a dword.
__device__ __forceinline__ uint32_t key_dword(uint32_t t, uint32_t dim) { return dim / 64 * 1024 + (dim / 16 % 4 * 16 + t) * 16 + dim % 16; }
__device__ __forceinline__ uint32_t value_dword(uint32_t t, uint32_t dim) { return dim / 64 * 1024 + (t / 4 * 16 + dim % 16) * 16 + dim / 16 % 4 * 4; }

// A run's place and scale.
struct Run {
    uint8_t *codes;  // of the block and kv head
    uint32_t dim, offset, count;
    bool raised;     // the codes before the run are to be moved to another scale
    float down, moved;
};
template <bool KEYS>
__device__ __forceinline__ Run run_of(const StoreArgs &a, size_t at, uint32_t dim, uint32_t offset, uint32_t count, float top, int before, int &e) {
    e = scale_exponent(top);
    if (offset > 0) e = max(e, min(max(before, LOWEST_EXPONENT), HIGHEST_EXPONENT));
    return {a.codes[KEYS ? 0 : 1] + at * (size_t(a.block_tokens) * SAETTA_HEAD_DIM), dim, offset, count, offset > 0 && e != before,
            power_of_two(-e), power_of_two(max(before - e, -126))};
}
// The lane's four dims of tokens t to t + 3 of the block, of which x holds those of the run.
template <bool KEYS>
__device__ __forceinline__ void put_tokens(const Run &r, uint32_t t, const float (&x)[4][4]) {
    const uint32_t token0 = t % UNIT_TOKENS;
    uint8_t *unit = r.codes + t / UNIT_TOKENS * UNIT_BYTES;
    auto rescaled = [&](uint32_t old) {
        float v[4];
        of_codes(old, v);
        return to_codes(v[0] * r.moved, v[1] * r.moved, v[2] * r.moved, v[3] * r.moved);
    };
    const uint32_t end = r.offset + r.count;
    // nothing of the four tokens is new, nor to be moved to another scale
    if (t >= end || (t + 4 <= r.offset && !r.raised)) return;
    if constexpr (KEYS) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t *p = reinterpret_cast<uint32_t *>(unit + key_dword(token0 + i, r.dim));
            if (t + i >= end || (t + i < r.offset && !r.raised)) continue;
            *p = t + i >= r.offset ? to_codes(x[i][0] * r.down, x[i][1] * r.down, x[i][2] * r.down, x[i][3] * r.down) : rescaled(*p);
        }
    } else {
        uint32_t fresh = 0, earlier = 0;  // bytes of tokens that are new; of tokens before them
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (t + i < r.offset) earlier |= 0xffu << (8 * i);
            else if (t + i < end) fresh |= 0xffu << (8 * i);
        }
        uint32_t old[4] = {0, 0, 0, 0};
        if (fresh != ~0u) {
#pragma unroll
            for (int d = 0; d < 4; d++) old[d] = *reinterpret_cast<const uint32_t *>(unit + value_dword(token0, r.dim + d));
        }
#pragma unroll
        for (int d = 0; d < 4; d++) {
            uint32_t value = to_codes(x[0][d] * r.down, x[1][d] * r.down, x[2][d] * r.down, x[3][d] * r.down);
            if (fresh != ~0u) value = (value & fresh) | ((r.raised ? rescaled(old[d]) : old[d]) & earlier) | (old[d] & ~(fresh | earlier));
            *reinterpret_cast<uint32_t *>(unit + value_dword(token0, r.dim + d)) = value;
        }
    }
}
__device__ __forceinline__ float largest(float top, const float (&x)[4]) {
#pragma unroll
    for (int d = 0; d < 4; d++) {
        const float m = fabsf(x[d]);
        top = m < __builtin_inff() ? fmaxf(top, m) : top;
    }
    return top;
}
template <int TYPE, bool KEYS>
__device__ __forceinline__ const typename Row<TYPE>::value *row_of_run(const StoreArgs &a, uint32_t token, uint32_t head, uint32_t dim) {
    const saetta_strided_rows &rows = a.x[KEYS ? 0 : 1];
    return static_cast<const typename Row<TYPE>::value *>(rows.data) + uint64_t(token) * rows.token_stride + head * rows.head_stride + dim;
}

// A run by the whole workgroup: a wave has four tokens of a unit, or of UNITS / 4 units, a lane four dims.
template <int TYPE, int UNITS, bool KEYS>
__device__ __forceinline__ void store_run(const StoreArgs &a, uint32_t token, uint32_t head, uint32_t block, uint32_t offset, uint32_t count) {
    constexpr uint32_t WAVES = store_waves(UNITS), AT_ONCE = WAVES / 4, EACH = UNITS / AT_ONCE;
    constexpr int which = KEYS ? 0 : 1;
    const uint32_t tid = threadIdx.x, wave = tid >> 6, dim = (tid & 63) * 4;
    // the run's token 0 sits at `offset`; token t of the block is row t - offset of the run
    const auto *x = row_of_run<TYPE, KEYS>(a, token, head, dim);
    const size_t at = size_t(block) * a.kv_heads + head;
    uint8_t *scale = a.scales[which] + at;
    const int before = int(*scale) - 127;
    auto first_of = [&](uint32_t u) { return (u * AT_ONCE + (wave >> 2)) * UNIT_TOKENS + (wave & 3) * 4; };
    float held[EACH][4][4];  // [unit][token][dim]
#pragma unroll
    for (uint32_t u = 0; u < EACH; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t t = first_of(u) + i;
#pragma unroll
            for (int d = 0; d < 4; d++) held[u][i][d] = 0.0f;
            if (t >= offset && t < offset + count) load_values<TYPE, 4>(x + uint64_t(t - offset) * a.x[which].token_stride, held[u][i]);
        }
    float top = 0.0f;
#pragma unroll
    for (uint32_t u = 0; u < EACH; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = largest(top, held[u][i]);
    top = group_reduce<64>(top, MaxOp());
    __shared__ float tops[WAVES];
    __syncthreads();  // the last run's have been read
    if ((tid & 63) == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) top = fmaxf(top, tops[w]);
    int e;
    const Run run = run_of<KEYS>(a, at, dim, offset, count, top, before, e);
#pragma unroll
    for (uint32_t u = 0; u < EACH; u++) put_tokens<KEYS>(run, first_of(u), held[u]);
    if (tid == 0) *scale = uint8_t(e + 127);  // (everyone has read it: there was a barrier since)
}

// A run of up to SHORT_RUN tokens by a wave.
template <int TYPE, bool KEYS>
__device__ __forceinline__ void store_short(const StoreArgs &a, uint32_t token, uint32_t head, uint32_t block, uint32_t offset, uint32_t count) {
    static_assert(SHORT_RUN == 4, "the tokens of a dword of values");
    constexpr int which = KEYS ? 0 : 1;
    const uint32_t lane = threadIdx.x & 63, dim = lane * 4;
    const auto *x = row_of_run<TYPE, KEYS>(a, token, head, dim);
    const size_t at = size_t(block) * a.kv_heads + head;
    uint8_t *scale = a.scales[which] + at;
    const int before = int(*scale) - 127;
    float held[SHORT_RUN][4], top = 0.0f;
#pragma unroll
    for (uint32_t j = 0; j < SHORT_RUN; j++) {
#pragma unroll
        for (int d = 0; d < 4; d++) held[j][d] = 0.0f;
        if (j < count) load_values<TYPE, 4>(x + uint64_t(j) * a.x[which].token_stride, held[j]);
    }
#pragma unroll
    for (uint32_t j = 0; j < SHORT_RUN; j++) top = largest(top, held[j]);
    top = group_reduce<64>(top, MaxOp());
    int e;
    const Run run = run_of<KEYS>(a, at, dim, offset, count, top, before, e);
    for (uint32_t t = run.raised ? 0 : offset & ~3u; t < offset + count; t += 4) {
        float y[4][4];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int d = 0; d < 4; d++) {
                const uint32_t j = t + i - offset;
                y[i][d] = j == 0 ? held[0][d] : j == 1 ? held[1][d] : j == 2 ? held[2][d] : held[3][d];
            }
        put_tokens<KEYS>(run, t, y);
    }
    if (lane == 0) *scale = uint8_t(e + 127);
}

// A workgroup looks at up to 64 tokens and takes the runs that begin there: the short ones a wave each, then the others one after the other.
template <int TYPE, int UNITS>
__global__ __launch_bounds__(64 * store_waves(UNITS)) void paged_store_kernel(StoreArgs a) {
    constexpr uint32_t BT = UNITS * UNIT_TOKENS, WAVES = store_waves(UNITS), TOKENS = lane_tokens(UNITS);
    const uint32_t head = blockIdx.y >> 1, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Lane i: slot of token token_of(i); whether a run begins there: what is before it in the call is in another block, or not the slot before;
    // the tokens that follow it in the block, slot by slot, up to SHORT_RUN.
    // (Every wave by itself: no barrier.)
    // The i-th token of TOKENS tokens is `step` workgroups further than the first: single tokens one behind the other are everyone's, and the blocks that a long
    // run fills are neighbours'.  (All by a workgroup: 64 single tokens of a step with room for 2048 47 us; now 5.)
    const uint32_t step = max(gridDim.x / TOKENS, 1u);
    auto token_of = [&](uint32_t i) { return (blockIdx.x + TOKENS * gridDim.x - i * step) % gridDim.x * TOKENS + i; };
    uint32_t slot = ~0u, follow = 0;
    bool begins = false;
    const uint32_t t = token_of(lane);
    if (lane < TOKENS && t < a.tokens) {
        slot = uint32_t(a.slots[t]);
        const uint32_t prior = t > 0 ? uint32_t(a.slots[t - 1]) : ~0u;
        uint32_t next[SHORT_RUN];
#pragma unroll
        for (uint32_t j = 0; j < SHORT_RUN; j++) next[j] = uint32_t(a.slots[min(t + 1 + j, a.tokens - 1)]);
        begins = slot / BT < a.blocks && (slot % BT == 0 || t == 0 || prior != slot - 1);  // (-1 is in no block)
        bool on = true;
#pragma unroll
        for (uint32_t j = 0; j < SHORT_RUN; j++) {
            on = on && slot % BT + 1 + j < BT && t + 1 + j < a.tokens && next[j] == slot + 1 + j;
            follow += on;
        }
    }
    const uint64_t all_runs = __ballot(begins), long_runs = __ballot(begins && follow >= SHORT_RUN);
    uint32_t turn = 0;
    for (uint64_t runs = all_runs & ~long_runs; runs; runs &= runs - 1, turn++) {
        if (turn % WAVES != wave) continue;
        const uint32_t i = uint32_t(__builtin_ctzll(runs)), token = token_of(i), from = __builtin_amdgcn_readlane(slot, i), count = 1 + __builtin_amdgcn_readlane(follow, i);
        if (blockIdx.y & 1) store_short<TYPE, false>(a, token, head, from / BT, from % BT, count);
        else store_short<TYPE, true>(a, token, head, from / BT, from % BT, count);
    }
    for (uint64_t runs = long_runs; runs; runs &= runs - 1) {
        const uint32_t i = uint32_t(__builtin_ctzll(runs)), token = token_of(i), from = __builtin_amdgcn_readlane(slot, i);
        const uint32_t block = from / BT, offset = from % BT;
        // the tokens that follow it in the block: up to 64 at a time
        uint32_t count = 1;
        for (uint32_t j0 = 1; j0 < BT - offset; j0 += 64) {
            const uint32_t j = j0 + lane;
            const bool follows = j < BT - offset && uint64_t(token) + j < a.tokens && uint32_t(a.slots[token + j]) == from + j;
            const uint64_t all = __ballot(follows);
            const uint32_t n = all == ~0ull ? 64 : uint32_t(__builtin_ctzll(~all));
            count += n;
            if (n < 64) break;
        }
        if (blockIdx.y & 1) store_run<TYPE, UNITS, false>(a, token, head, block, offset, count);
        else store_run<TYPE, UNITS, true>(a, token, head, block, offset, count);
    }
}

struct GatherArgs {
    const uint8_t *codes[2], *scales[2];
    const int32_t *slots;
    void *out[2];
    uint32_t blocks, block_tokens, kv_heads, tokens;
};

// A workgroup takes 16 slots of one kv head, keys or values: a wave a slot at a time, a lane four dims, so that a store is a whole row.
// Where the slots lie in two units at most (16 that follow each other do), the units come through LDS by whole kilobytes, for values are stored
// four tokens to a dword; else a lane reads its bytes where they are.  32768 tokens, f16, 2 kv heads: 19 to 20 us, 5.2 TB/s of what is read and written.  (A
// lane's bytes straight from memory: 42 us.  Rows that keep a place in the caches on their way out: 29 where every call has other data, and who reads them
// next takes as long either way.)
constexpr uint32_t GATHER_SLOTS = 16;
template <int TYPE>
__global__ __launch_bounds__(256) void paged_gather_kernel(GatherArgs a) {
    typedef typename Row<TYPE>::value V;
    __shared__ __attribute__((aligned(16))) uint8_t units[2][UNIT_BYTES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, head = blockIdx.y >> 1, which = blockIdx.y & 1;
    if (a.out[which] == nullptr) return;
    const uint64_t row0 = uint64_t(blockIdx.x) * GATHER_SLOTS;
    // lane i (< 16): slot i; those that are not there take no part
    uint32_t slot = ~0u;
    if (lane < GATHER_SLOTS && row0 + lane < a.tokens) slot = uint32_t(a.slots[row0 + lane]);
    const uint64_t there = __ballot(slot / a.block_tokens < a.blocks);
    if (there == 0) return;
    const uint32_t first = __builtin_amdgcn_readlane(slot, __builtin_ctzll(there)) / UNIT_TOKENS, last = __builtin_amdgcn_readlane(slot, 63 - __builtin_clzll(there)) / UNIT_TOKENS;
    const bool near = (__ballot(slot / UNIT_TOKENS == first || slot / UNIT_TOKENS == last) & there) == there;
    auto row_of = [&](uint32_t unit) { return size_t(unit / (a.block_tokens / UNIT_TOKENS)) * a.kv_heads + head; };
    auto codes_of = [&](uint32_t unit) { return a.codes[which] + row_of(unit) * (size_t(a.block_tokens) * SAETTA_HEAD_DIM) + unit % (a.block_tokens / UNIT_TOKENS) * UNIT_BYTES; };
    if (near) {
        const uint4 x = *reinterpret_cast<const uint4 *>(codes_of(first) + tid * 16), y = *reinterpret_cast<const uint4 *>(codes_of(last) + tid * 16);
        *reinterpret_cast<uint4 *>(units[0] + tid * 16) = x, *reinterpret_cast<uint4 *>(units[1] + tid * 16) = y;
    }
    __syncthreads();
    const uint32_t dim = lane * 4;
#pragma unroll
    for (uint32_t k = 0; k < GATHER_SLOTS / 4; k++) {
        const uint32_t i = wave * (GATHER_SLOTS / 4) + k;
        if (!(there >> i & 1)) continue;
        const uint32_t from = __builtin_amdgcn_readlane(slot, i), unit = from / UNIT_TOKENS, t = from % UNIT_TOKENS;
        const float scale = power_of_two(int(a.scales[which][row_of(unit)]) - 127);
        auto bytes = [&](const uint8_t *p) {
            if (which == 0) return *reinterpret_cast<const uint32_t *>(p + key_dword(t, dim));
            p += value_dword(t, dim) + t % 4;
            return uint32_t(p[0]) | uint32_t(p[16]) << 8 | uint32_t(p[32]) << 16 | uint32_t(p[48]) << 24;
        };
        float x[4];
        of_codes(near ? bytes(units[unit == first ? 0 : 1]) : bytes(codes_of(unit)), x);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] *= scale;
        store_values<TYPE, 4, true>(static_cast<V *>(a.out[which]) + ((row0 + i) * a.kv_heads + head) * SAETTA_HEAD_DIM + dim, x);
    }
}

template <int TYPE, int UNITS>
void launch_store(hipStream_t stream, const StoreArgs &a) {
    const uint32_t sides = a.kv_heads * 2;
    uint32_t groups = STORE_GROUPS / sides < a.tokens ? STORE_GROUPS / sides : a.tokens;
    const uint32_t least = (a.tokens + lane_tokens(UNITS) - 1) / lane_tokens(UNITS);
    if (groups < least) groups = least;
    launch(paged_store_kernel<TYPE, UNITS>, dim3(groups, sides), dim3(64 * store_waves(UNITS)), 0, stream, a);
}
template <int TYPE>
void launch_store(hipStream_t stream, const StoreArgs &a) {
    switch (a.block_tokens) {
        case 16: return launch_store<TYPE, 1>(stream, a);
        case 32: return launch_store<TYPE, 2>(stream, a);
        case 64: return launch_store<TYPE, 4>(stream, a);
        default: return launch_store<TYPE, 8>(stream, a);
    }
}

}  // namespace

int setup_paged_cache() { return load_kernel(reinterpret_cast<const void *>(paged_gather_kernel<SAETTA_F16>)); }

}  // namespace saetta

using namespace saetta;

extern "C" int saetta_paged_store(saetta_stream_t stream, int type, saetta_strided_rows keys, saetta_strided_rows values,
                                  const int32_t *slots, saetta_paged_cache cache, uint32_t tokens) {
    SAETTA_REQUIRE(type == SAETTA_F32 || type == SAETTA_F16 || type == SAETTA_BF16, SAETTA_E_BITS, "paged_store: type %d (f32, f16 or bf16)", type);
    SAETTA_REQUIRE(tokens == 0 || (keys.data && values.data && slots), SAETTA_E_NULL, "paged_store: null buffer");
    if (int rc = check_cache(cache, "paged_store")) return rc;
    SAETTA_REQUIRE(aligned(slots, 4) && rows_aligned(keys, type) && rows_aligned(values, type), SAETTA_E_ALIGN,
                   "paged_store: keys and values must be 16-byte aligned, with strides of multiples of 16 bytes");
    SAETTA_REQUIRE(tokens <= MOST_TOKENS, SAETTA_E_SHAPE, "paged_store: %u tokens (at most 2^28 - 32)", tokens);
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
    SAETTA_REQUIRE(tokens == 0 || slots, SAETTA_E_NULL, "paged_gather: null slots");
    if (int rc = check_cache(cache, "paged_gather")) return rc;
    SAETTA_REQUIRE(aligned(slots, 4) && aligned(keys, 16) && aligned(values, 16), SAETTA_E_ALIGN, "paged_gather: keys and values must be 16-byte aligned");
    SAETTA_REQUIRE(tokens <= MOST_TOKENS, SAETTA_E_SHAPE, "paged_gather: %u tokens (at most 2^28 - 32)", tokens);
    if (int rc = ensure_device()) return rc;
    if (tokens == 0 || (!keys && !values)) return SAETTA_OK;
    const GatherArgs a = {{cache.keys, cache.values}, {cache.key_scales, cache.value_scales}, slots, {keys, values},
                          cache.blocks, cache.block_tokens, cache.kv_heads, tokens};
    const dim3 grid((tokens + GATHER_SLOTS - 1) / GATHER_SLOTS, cache.kv_heads * 2);
    if (type == SAETTA_F32) launch(paged_gather_kernel<SAETTA_F32>, grid, dim3(256), 0, as_stream(stream), a);
    else if (type == SAETTA_F16) launch(paged_gather_kernel<SAETTA_F16>, grid, dim3(256), 0, as_stream(stream), a);
    else launch(paged_gather_kernel<SAETTA_BF16>, grid, dim3(256), 0, as_stream(stream), a);
    return launch_status("paged_gather");
}
