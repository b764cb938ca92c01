// Attention of a step's new tokens over a cache in blocks for several requests.
//
// For row i of request r, at position p = kv_lens[r] - n + i, and q head h over kv head h / group:
//     out = sum_t 2^(s_t) v_t / sum_t 2^(s_t) [* sigmoid(gate)],  s_t = log2(e) scale (q . k_t),  t = 0 .. p.
// The cache holds codes a, b and exponents: k_t = 2^ek a_t, v_t = 2^ev b_t, one ek and ev per block and kv head.  With ev = held + rest, held
// of -15..7,
//     x_t = log2(e) scale 2^ek (q . a_t) + rest,   w_t = 2^(x_t - M),
// out = sum w_t (2^held b_t) / sum w_t 2^-rest.  The matrix cores see codes of keys, which f16 and bf16 hold exactly, and codes of values times 2^held, which
// f16 holds exactly too (from 2^-9 * 2^-15, its least number, to 448 * 2^7): where a block's largest value is 0.014 to 57344 the weights are
// the softmax's own, and only past that is what is left of the exponent an addend of the score.  (All of it as an addend, a block that is loud in one dim
// took the weights of blocks 2^34 quieter out of f16's range in every dim.)
// M follows the running maximum, 7 to 15 below it, so that the largest weight is 2^7 to 2^15.  Only w_t is rounded (to f16, as operand of the second product:
// by up to 2^-11 of it, or 2^-25 where it is below 2^-14, which is 2^-32 of the largest at most; with M at the maximum 2^-25, and 131072 keys just below that were
// 0.4 % of a row.  Tiles of up to 16 rows add what was rounded off); the sums are f32, that of the weights of unrounded ones.
//
// The three kernels: paged_split_kernel deals rows and keys out as items from the lengths; the attention kernel, one
// workgroup to an item and kv head, paged_few_kernel for tiles of up to 64 rows and paged_chunk_kernel for tiles of
// 256; paged_merge_kernel where a tile's keys were taken in parts.
//
// Both attention kernels compute S^T = K Q^T and O^T += V^T P^T: a lane owns one query row (column), the running
// maximum and sum are its own, and the probabilities go from the accumulators of the first product into the operand of the
// second as they lie.  The cache's order of bytes is that of the operands: a load of a wave is one contiguous kilobyte.
#include "common.hpp"
#include "lanes.hpp"
#include "paged_device.hpp"

namespace saetta {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4_ __attribute__((ext_vector_type(4)));
typedef _Float16 half2_ __attribute__((ext_vector_type(2)));
typedef __bf16 brain8 __attribute__((ext_vector_type(8)));
typedef __bf16 brain2 __attribute__((ext_vector_type(2)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int DIM = SAETTA_HEAD_DIM;
#include "prefill_stream.hpp"  // scores_block, stream_block_alone, settle
constexpr float NO_SCORE = -__builtin_inff();    // of a key that a row does not see
constexpr float NO_MAXIMUM = -1e30f;             // where nothing was seen: 2^(NO_SCORE - NO_MAXIMUM) is 0
constexpr float TAU = 8.0f;                      // M is raised only when the maximum has risen by this many powers of two
constexpr float TOP = 7.0f;                      // the maximum less M as M is raised: with TAU the largest weight is 2^15, in f16's range
constexpr int LOWEST_HELD = -15, HIGHEST_HELD = 7;  // of a values' exponent, what their conversion to f16 takes
constexpr uint32_t STEP_KEYS = 32;               // keys of a step: two units
constexpr uint32_t FEW_ROWS = 16, CHUNK_ROWS = 256;  // FEW_ROWS: of a group of columns; a tile of few rows has 1, 2 or 4 groups
constexpr int FEW_WAVES = 4, CHUNK_WAVES = 8;

// ---- what is dealt out -------------------------------------------------------------------------------------------

// Rows of a request and keys that a workgroup takes.
struct alignas(16) Item {
    uint32_t request, row0, tokens;  // rows of q from row0 on
    int32_t pos0;                    // position of the first of them
    uint32_t key0, key1;             // keys that are taken (up to what the last row sees)
    uint32_t slot;                   // where its sums go, if the tile's keys are taken in parts; of a tile in parts, its first part's
    uint32_t parts;                  // of the tile
};
struct alignas(16) SplitHead {
    uint32_t items, tiles;  // items dealt out; tiles in parts, which are joined afterwards
    uint32_t unused[2];
};

struct Shape {
    uint32_t group, tile_tokens, tile_rows;
    uint32_t columns;  // groups of FEW_ROWS rows of the kernel for few rows; 0: chunks
    uint32_t target;  // items that the device takes at once
    uint32_t most_items, most_tiles, most_joined, slots;
};
Shape shape_of(const saetta_paged_attn_params &p, uint32_t requests) {
    Shape s;
    s.group = p.heads / p.kv_heads;
    const uint64_t rows = uint64_t(p.rows) * s.group;
    s.columns = rows <= FEW_ROWS ? 1 : rows <= 2 * FEW_ROWS ? 2 : rows <= 4 * FEW_ROWS ? 4 : 0;
    const bool few = s.columns > 0;
    s.tile_rows = few ? s.columns * FEW_ROWS : CHUNK_ROWS;
    s.tile_tokens = few ? p.rows : CHUNK_ROWS / s.group;
    const uint32_t workgroups = cu_count() * (s.columns == 1 ? 2 : 1);
    s.target = workgroups / p.kv_heads ? workgroups / p.kv_heads : 1;
    s.most_tiles = few ? requests : p.tokens / s.tile_tokens + requests;
    // With parts of total / target no more than `target` tiles have more than one, and their parts are 2 * target at most
    s.most_items = s.most_tiles + s.target;
    s.most_joined = s.target < s.most_tiles ? s.target : s.most_tiles;
    s.slots = 2 * s.target;
    return s;
}

struct SplitArgs {
    saetta_paged_batch batch;
    SplitHead *head;
    Item *items, *tiles;
    uint32_t tile_tokens, target, most_items, most_joined, slots, tokens, rows;
    uint32_t few, granule, least, extra, few_tokens, half_tokens;  // (granule: a power of two)
};

// What an item of a chunk costs besides its keys, in keys (15 us of a workgroup, and its sums' way through memory): seven prompts of 147 to
// 1645 tokens, attention and merge, 96 us with 0, 94 with 256, 92 with 512, 104 with 768; a chunk beside drafts the same with all.
constexpr uint32_t CHUNK_EXTRA = 512;
// Keys that a part has at least.  32 tokens at 992 41 us with 512, 30 with 256, 25 with 128 and 64; 300 at 0 37, 37, 32, 30; 32 at 8000 46, 41, 41, 49.
constexpr uint32_t LEAST_KEYS = 128;

constexpr uint32_t SIZES = 64;  // classes of items by what they cost

// A request as the split sees it.
struct Work {
    uint32_t row0, tokens, tiles;
    int32_t pos0;
};
__device__ __forceinline__ Work work_of(const SplitArgs &a, uint32_t r) {
    Work w = {0, 0, 0, 0};
    if (r >= a.batch.requests) return w;
    const uint32_t start = min(a.batch.query_starts[r], a.tokens), end = min(a.batch.query_starts[r + 1], a.tokens);
    const uint32_t n = end > start ? end - start : 0;
    w.row0 = start, w.tokens = a.few ? min(n, a.rows) : n;
    w.pos0 = int32_t(min(a.batch.kv_lens[r], 0x7fffffffu)) - int32_t(n);
    w.tiles = (w.tokens + a.tile_tokens - 1) / a.tile_tokens;
    return w;
}
// Tile `tile` of it, whole.
__device__ __forceinline__ Item tile_of(const SplitArgs &a, const Work &w, uint32_t r, uint32_t tile) {
    Item item;
    const uint32_t first = tile * a.tile_tokens;
    item.request = r, item.row0 = w.row0 + first, item.tokens = min(a.tile_tokens, w.tokens - first);
    item.pos0 = w.pos0 + int32_t(first);
    item.key0 = 0, item.key1 = min(uint32_t(max(item.pos0 + int32_t(item.tokens), 0)), a.batch.max_blocks * a.batch.block_tokens);
    item.slot = 0, item.parts = 1;
    return item;
}

// x summed over the threads before this one; `all`: over all of them.  (All threads; `waves` is free again on return.)
template <uint32_t SPLIT_THREADS>
__device__ __forceinline__ uint32_t before_this(uint32_t x, uint32_t *waves, uint32_t &all) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t through = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t other = __shfl_up(through, d);
        if (lane >= uint32_t(d)) through += other;
    }
    if (lane == 63) waves[wave] = through;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < SPLIT_THREADS / 64; w++) {
        if (w < wave) before += waves[w];
        all += waves[w];
    }
    __syncthreads();
    return before + through - x;
}

// Deals the work out so that the workgroups that run at once end together.  What a key of a tile costs is one of three numbers: a chunk's tile of
// at most half the rows keeps half the waves and takes 6 / 8 of the time, one of up to 64 rows is taken as few rows are, by the memory's rate.  A tile that costs more than total / target is cut into parts of that
// and a rest; the items go out from the dearest class to the cheapest, so that who ends early takes what is small.  (One workgroup: a sum over the
// tiles, a count of the classes, and the items themselves; the tiles by turns over its threads.  The places of the items in a class and of the
// parts' sums follow from atomic counts, in any order: what is computed does not depend on them.)  Latency: 5 us for one request, 7 for 48, 8.4 for a
// chunk beside 30 drafts, once a step.
template <uint32_t SPLIT_THREADS>
__global__ __launch_bounds__(SPLIT_THREADS) void paged_split_kernel(SplitArgs a) {
    __shared__ uint32_t waves[SPLIT_THREADS / 64], starts[SPLIT_THREADS], ends[SPLIT_THREADS], classes[SIZES], slots_there, tiles_there;
    __shared__ unsigned long long total, items_there;
    __shared__ Item cut[SPLIT_THREADS];
    const uint32_t tid = threadIdx.x, requests = a.batch.requests;
    if (tid < SIZES) classes[tid] = 0;
    if (tid == 0) slots_there = tiles_there = 0, total = items_there = 0;
    __syncthreads();

    // Requests by rounds of as many as there are threads, their tiles by rounds too: f(a tile of this thread's, or one of no tokens), all threads
    // alike.  Where one round holds all (as a rule) the tile is found once.
    bool found = false;
    Item mine;
    mine.tokens = 0;  // (and remains so where no request has a new token)
    auto for_tiles = [&](auto f) {
        if (found) return f(mine);
        uint32_t most = a.most_items - a.target;  // as many tiles as there can be, whatever the starts say
        for (uint32_t r0 = 0; r0 < requests; r0 += SPLIT_THREADS) {
            uint32_t all;
            const uint32_t tiles = work_of(a, r0 + tid).tiles, before = before_this<SPLIT_THREADS>(tiles, waves, all), n = min(SPLIT_THREADS, requests - r0);
            all = min(all, most), most -= all;
            starts[tid] = before;
            __syncthreads();
            for (uint32_t k0 = 0; k0 < all; k0 += SPLIT_THREADS) {
                const uint32_t k = k0 + tid;
                mine.tokens = 0;
                if (k < all) {
                    const uint32_t i = last_at_most(starts, n, k);
                    mine = tile_of(a, work_of(a, r0 + i), r0 + i, k - starts[i]);
                }
                f(mine);
            }
            found = requests <= SPLIT_THREADS && all <= SPLIT_THREADS;
            __syncthreads();  // `starts` may be written again
        }
    };
    // FEW: a chunk of 1500 tokens beside 30 drafts 283 us with 3, 267 with 4, 272 with 5.  HALF: seven prompts 92 us with 4, 79 with 5, 74 with 6 and 7.
    constexpr uint32_t FEW = 4, HALF = 6, WHOLE = 8;
    auto price = [&](const Item &tile) { return tile.tokens <= a.few_tokens ? FEW : tile.tokens <= a.half_tokens ? HALF : WHOLE; };

    // a number of every thread, added up into `into`, which is 0
    auto add_up = [&](unsigned long long x, unsigned long long *into) {
#pragma unroll
        for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d);
        if ((tid & 63) == 0 && x) atomicAdd(into, x);
        __syncthreads();
    };
    unsigned long long sum = 0;
    for_tiles([&](const Item &tile) { sum += tile.tokens ? static_cast<unsigned long long>(tile.key1) * price(tile) : 0; });
    add_up(sum, &total);
    // what a part costs at most, and its keys
    unsigned long long fair = max(total / a.target + 1, static_cast<unsigned long long>(a.least) * 8);
    auto length_at = [&](unsigned long long keys) {
        keys += a.granule;
        return uint32_t(keys > 0x7fffffffu ? 0x7fffffffu : keys) & ~(a.granule - 1);
    };
    uint32_t few_length = length_at(fair / FEW), half_length = length_at(fair / HALF), whole_length = length_at(fair / WHOLE);
    // (sums: as three choices of a variable the compiler puts the tile in memory, and the kernel takes half as long again)
    auto length_of = [&](const Item &tile) {
        return whole_length + (tile.tokens <= a.half_tokens ? half_length - whole_length : 0) + (tile.tokens <= a.few_tokens ? few_length - half_length : 0);
    };
    if (a.extra) {
        // An item costs `extra` keys besides its own (its start and end, its sums through memory): a share of as many items as there now are
        unsigned long long items = 0;
        for_tiles([&](const Item &tile) { items += tile.tokens ? max((tile.key1 + length_of(tile) - 1) / length_of(tile), 1u) : 0; });
        add_up(items, &items_there);
        if (items_there > a.target) fair += (items_there - a.target) * 8 * a.extra / a.target;
        few_length = length_at(fair / FEW), half_length = length_at(fair / HALF), whole_length = length_at(fair / WHOLE);
    }
    const float per_class = float(SIZES) / float(fair + 8ull * a.granule);
    auto class_of = [&](uint32_t keys, uint32_t price) { return SIZES - 1 - min(uint32_t(float(keys) * float(price) * per_class), SIZES - 1); };
    for_tiles([&](const Item &tile) {
        if (!tile.tokens) return;
        const uint32_t length = length_of(tile), whole = tile.key1 / length, rest = tile.key1 - whole * length;
        if (whole) atomicAdd(&classes[class_of(length, price(tile))], whole);
        if (rest || !whole) atomicAdd(&classes[class_of(rest, price(tile))], 1u);
    });
    __syncthreads();
    if (tid < 64) {  // where each class begins
        static_assert(SIZES == 64, "a lane a class");
        const uint32_t n = classes[tid];
        uint32_t through = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const uint32_t other = __shfl_up(through, d);
            if (tid >= uint32_t(d)) through += other;
        }
        classes[tid] = through - n;
        if (tid == 63) a.head->items = min(through, a.most_items);
    }
    __syncthreads();
    // the items: a round's tiles in LDS, their parts over all threads
    for_tiles([&](Item tile) {
        const uint32_t length = tile.tokens ? length_of(tile) : 1;
        tile.parts = !tile.tokens ? 0 : tile.key1 > length ? (tile.key1 + length - 1) / length : 1;
        if (tile.parts > 1) {
            tile.slot = atomicAdd(&slots_there, tile.parts);
            const uint32_t t = atomicAdd(&tiles_there, 1u);
            if (t < a.most_joined) a.tiles[t] = tile;
        }
        uint32_t all;
        ends[tid] = before_this<SPLIT_THREADS>(tile.parts, waves, all);
        cut[tid] = tile;
        __syncthreads();
        for (uint32_t k = tid; k < all; k += SPLIT_THREADS) {
            const uint32_t i = last_at_most(ends, SPLIT_THREADS, k);
            Item item = cut[i];
            const uint32_t each = length_of(item), p = k - ends[i];
            item.key0 = p * each, item.key1 = min(item.key1, item.key0 + each), item.slot += p;
            const uint32_t where = atomicAdd(&classes[class_of(item.key1 - item.key0, price(item))], 1u);
            if (where < a.most_items) a.items[where] = item;
        }
        __syncthreads();
    });
    if (tid == 0) a.head->tiles = min(tiles_there, a.most_joined);
}

// ---- the attention kernels ----------------------------------------------------------------------------------------

// Rows whose strides fit 32 bits: a lane's address is two multiply-adds (with 64 bits to both factors it was a dozen instructions of a quarter of the
// rate, half the time of a chunk tile's end).
struct Rows {
    void *data;
    uint32_t token_stride, head_stride;
};
template <class V>
__device__ __forceinline__ V *row_at(const Rows &r, uint32_t token, uint32_t head) {
    return static_cast<V *>(r.data) + uint64_t(token) * r.token_stride + uint64_t(head) * r.head_stride;
}

struct AttnArgs {
    Rows q, gate, out;
    saetta_paged_cache cache;
    const int32_t *block_table;
    const SplitHead *head;
    const Item *items;
    float *part_o;   // [slot][kv head][tile rows][256], relative to M
    float *part_ml;  // [slot][kv head][tile rows][M, sum]
    uint32_t requests, max_blocks, tokens, group, group_shift, block_shift, slots, tile_tokens;
    float scale;
};

// Codes of one dword as four halves, times a power of two.
__device__ __forceinline__ u32x2 halves_of(uint32_t w, float scale) {
    const half2_ a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
template <int TYPE>
__device__ __forceinline__ u32x2 operands_of(uint32_t w) {
    if constexpr (TYPE == SAETTA_F16) return halves_of(w, 1.0f);
    const brain2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true);
    return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}
template <int TYPE>
__device__ __forceinline__ u32x4 operands_of(uint32_t w0, uint32_t w1) {
    const u32x2 a = operands_of<TYPE>(w0), b = operands_of<TYPE>(w1);
    return u32x4{a.x, a.y, b.x, b.y};
}
template <int TYPE>
__device__ __forceinline__ floatx4 product16(u32x4 a, u32x4 b, floatx4 c) {
    if constexpr (TYPE == SAETTA_F16) return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(brain8, a), __builtin_bit_cast(brain8, b), c, 0, 0, 0);
}
template <int TYPE>
__device__ __forceinline__ floatx16 product32(u32x4 a, u32x4 b, floatx16 c) {
    if constexpr (TYPE == SAETTA_F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(brain8, a), __builtin_bit_cast(brain8, b), c, 0, 0, 0);
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const half2_ h = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, h);
}
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.4426950408889634f)); }

// Where a unit of 16 tokens lies and what its codes are scaled by.  Units that are not there (no block, or not one of the
// cache) are read from the cache's first block and masked.
struct Unit {
    uint32_t block;     // row of [blocks][kv_heads]; of the first block where there is none
    uint32_t scales;    // 127 + ek | (127 + ev) << 8 | there << 16
};
// Units that a workgroup keeps in LDS: unit u at u % WINDOW.  From `end` on there are none.
constexpr uint32_t WINDOW = 512;
__device__ __forceinline__ Unit find_unit(const AttnArgs &a, uint32_t request, uint32_t head, uint32_t u, uint32_t end) {
    const uint32_t entry = u >> (a.block_shift - 4);
    uint32_t block = ~0u;
    if (u < end && entry < a.max_blocks) block = uint32_t(a.block_table[size_t(request) * a.max_blocks + entry]);
    const bool there = block < a.cache.blocks;
    return {(there ? block : 0) * a.cache.kv_heads + head, uint32_t(there) << 16};
}
__device__ __forceinline__ uint32_t find_scales(const AttnArgs &a, const Unit &u) {
    return u.scales | uint32_t(a.cache.key_scales[u.block]) | uint32_t(a.cache.value_scales[u.block]) << 8;
}
// (exponents as the store writes them: what else a byte says would make scores no numbers)
__device__ __forceinline__ float key_scale(uint32_t scales) { return power_of_two(min(max(int(scales & 0xff) - 127, LOWEST_EXPONENT), HIGHEST_EXPONENT)); }
// ev of a unit's values, in two: what their conversion takes, and the rest, the score's.
struct ValueExponent {
    int held, rest;
};
__device__ __forceinline__ ValueExponent value_exponent(uint32_t scales) {
    const int e = min(max(int(scales >> 8 & 0xff) - 127, LOWEST_EXPONENT), HIGHEST_EXPONENT), held = min(max(e, LOWEST_HELD), HIGHEST_HELD);
    return {held, e - held};
}

// An item that the split has made for these buffers.  (A split of other parameters is not followed out of them.)  (No branches: the
// loads go out together.)
__device__ __forceinline__ bool item_ok(const AttnArgs &a, const Item &item, uint32_t slots) {
    return int(item.request < a.requests) & int(item.tokens > 0) & int(item.tokens <= a.tile_tokens) & int(item.row0 <= a.tokens) &
           int(item.tokens <= a.tokens - min(item.row0, a.tokens)) & int(item.key1 <= a.max_blocks << a.block_shift) &
           int((int(item.parts == 1) | (int(item.slot < a.slots) & int(slots <= a.slots - min(item.slot, a.slots)))) != 0);
}

// Bytes of a dword of four tokens' values that are NaN, as 0x80 in each.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// Bytes of the first n of four tokens.
__device__ __forceinline__ uint32_t first_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; }

// A dword of four tokens' values of one dim, cleared where no row may see it: from key `limit` on what a block happens to
// hold, and NaN from key `all` on, where the tile's first rows end (0 * NaN would reach rows that do not see the token; nan_from
// [256] keeps the first such key of a dim, and the rows that do see it become NaN at the end).
__device__ __forceinline__ uint32_t clean_values(uint32_t w, uint32_t key, uint32_t limit, uint32_t all, uint32_t dim, uint32_t *nan_from) {
    w &= first_bytes(int(limit) - int(key));
    const uint32_t bad = nan_bytes(w) & ~first_bytes(int(all) - int(key));
    if (bad) {
        atomicMin(&nan_from[dim], key + (__builtin_ctz(bad) >> 3));
        w &= ~((bad >> 7) * 0xffu);
    }
    return w;
}

// out of a row's four dims
template <int TYPE>
__device__ __forceinline__ void put_row(const AttnArgs &a, uint32_t row, uint32_t head, uint32_t dim, float (&o)[4]) {
    typedef typename Row<TYPE>::value V;
    if (a.gate.data) {
        float g[4];
        load_values<TYPE, 4>(row_at<const V>(a.gate, row, head) + dim, g);
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] *= sigmoid(g[i]);
    }
    store_values<TYPE, 4>(row_at<V>(a.out, row, head) + dim, o);
}

// Few rows (a call's, or a tile's of a chunk call): a workgroup of 4 waves walks an item's keys, every wave 32 of 128 at a time, straight from memory into registers, the
// keys of its next step on their way while this one's values are worked on, and the other way round.  Bound by memory: 16 KB a step of a
// wave, against 64 + 64 conversions of two codes and, a group of 16 rows (COLUMNS of them), 16 + 16 products.  Row l % 16 of a group is lane
// l's; the waves' sums are joined in LDS, a group after the other.  A wave looks up the places of the units of its next 32 steps by itself, a
// unit a lane: no barrier in the walk, and the scales, which only the scores want, come behind the first codes.
// One group is two workgroups to a CU; two have the registers of a SIMD to themselves; of four, two teams of four waves take two each over the
// same keys, whose codes the second team finds in the caches.  (The kernel for chunks, where most of a tile is empty, takes 102 to 108 us for 64 drafts of 3
// to 8 tokens at 4000, this one 49 to 69; four groups to a wave are more registers than there are: 353.)
// Measured, 8 q heads over each of 2 kv heads: a token of 8 requests at 131072 tokens, f16, 162 us, 6.6 TB/s of codes (a large copy reaches 4.9, read and
// written); of 48 requests at 330 to 30 thousand tokens, bf16, 56 us, 5.9 TB/s; of one at 517 tokens 7 to 8 us, the launch and three loads that wait for each other.
constexpr int few_threads(int columns) { return 64 * FEW_WAVES * (columns == 4 ? 2 : 1); }
constexpr uint32_t FEW_STEPS = 32;     // steps that a wave looks up at a time
constexpr int FEW_STRIDE = DIM + 4;    // floats of a row in LDS: neighbouring rows on other banks
// What the waves of a workgroup share.
template <int COLUMNS, int TEAMS, int TURNS>
struct FewShared {
    float sums[TURNS][FEW_ROWS][FEW_STRIDE];
    float ml[TURNS][FEW_ROWS][2];
    static constexpr bool IN_LDS = TEAMS * TURNS == 8 && TEAMS * COLUMNS > 1;  // the queries: two waves share the registers of a SIMD
    u32x4 queries[IN_LDS ? COLUMNS * TEAMS : 1][IN_LDS ? 8 : 1][IN_LDS ? 64 : 1];
};
// An item of up to COLUMNS * TEAMS groups by TEAMS teams of TURNS waves, COLUMNS groups to a wave; the parts' sums lie TILE rows apart.
template <int TYPE, int COLUMNS, int TEAMS, int TURNS, uint32_t TILE>
__device__ __forceinline__ void take_few(const AttnArgs &a, const Item &item, uint32_t kv, FewShared<COLUMNS, TEAMS, TURNS> &shared, uint32_t *nan_from) {
    typedef typename Row<TYPE>::value V;
    constexpr int TILE_COLUMNS = COLUMNS * TEAMS;
    // A wave with one group multiplies what is rounded off its weights too, as another f16 (2^-22 of a weight, or 2^-32 of the largest, is left): the matrix cores are idle
    // there for most of the time.  8 requests at 131072 171.8 -> 172.7 us with split and merge, four layers of 48 ragged 244 -> 246, of 64 requests of two tokens at 4000
    // 213 -> 215.  With two groups it would be 223 -> 236 for three tokens, with four 333 -> 349 for five.
    constexpr bool BOTH_HALVES = COLUMNS == 1;
    constexpr uint32_t WAVES = TEAMS * TURNS;
    auto &sums = shared.sums;
    auto &ml = shared.ml;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t col = lane & 15, quarter = lane >> 4;
    const uint32_t team = wave / TURNS, turn = wave % TURNS;  // the wave's groups; its keys
    const uint32_t rows = item.tokens << a.group_shift;  // of the tile that are there
    for (uint32_t i = tid; i < DIM; i += 64 * WAVES) nan_from[i] = ~0u;

    const size_t block_bytes = size_t(DIM) << a.block_shift;
    const uint32_t unit_shift = a.block_shift - 4, unit_mask = (1u << unit_shift) - 1;
    const uint32_t end_unit = (item.key1 + UNIT_TOKENS - 1) / UNIT_TOKENS;
    uint32_t first = item.key0 / UNIT_TOKENS + 2 * turn;  // the wave's first unit; its steps are 2 * TURNS units apart
    // Lane 2 i + j: unit j of step i, its row of [blocks][kv heads] (of block 0 where there is none) and whether there is one.
    uint32_t place = 0, scales = 0;
    auto look_up = [&] {
        const uint32_t unit = first + (lane >> 1) * (2 * TURNS) + (lane & 1), entry = unit >> unit_shift;
        uint32_t block = ~0u;
        if (unit < end_unit && entry < a.max_blocks) block = uint32_t(a.block_table[size_t(item.request) * a.max_blocks + entry]);
        const bool there = block < a.cache.blocks;
        place = (there ? block : 0) * a.cache.kv_heads + kv;
        scales = uint32_t(there) << 16;
    };
    auto look_up_scales = [&] { scales |= uint32_t(a.cache.key_scales[place]) | uint32_t(a.cache.value_scales[place]) << 8; };
    u32x4 k[2][4], v[2][4];  // codes of a step: [unit][64 dims]
    // (One team's codes are read once, and between two steps of a model its weights go through the caches: marked as such, what is read keeps no
    // place there.  64 requests of 8000 tokens 93.4 -> 82.3 us, 48 ragged 63 -> 55, 16 of 2000 the same; where the last call left the codes in the caches
    // 41.8 -> 43.1, one of 517 6.3 -> 7.3, where 48 requests share all their 8000 tokens 30.6 -> 37.8.)
    auto fetch = [&](const uint8_t *codes, uint32_t step, u32x4 (&x)[2][4]) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t row = __builtin_amdgcn_readlane(place, 2 * step + i), unit = (first + step * (2 * TURNS) + i) & unit_mask;
            const uint8_t *at = codes + row * block_bytes + unit * UNIT_BYTES;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const u32x4 *from = reinterpret_cast<const u32x4 *>(at + j * 1024 + lane * 16);
                if constexpr (TEAMS == 1) x[i][j] = __builtin_nontemporal_load(from);
                else x[i][j] = *from;
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (on their way from here on, not where they are wanted)
    };
    uint32_t steps = first < end_unit ? (end_unit - first + 2 * TURNS - 1) / (2 * TURNS) : 0;  // that are left
    if (steps) {
        look_up();
        fetch(a.cache.keys, 0, k);
        look_up_scales();
    }

    // The queries: [group][64 dims][8 of 16].
    constexpr bool IN_LDS = FewShared<COLUMNS, TEAMS, TURNS>::IN_LDS;
    u32x4 q[IN_LDS ? 1 : COLUMNS][8];
    auto &q_lds = shared.queries;
    int32_t sees[COLUMNS];  // keys of this lane's rows
    auto row_of = [&](uint32_t g) { return min(g * FEW_ROWS + col, rows - 1); };
    auto q_of = [&](uint32_t g, int i) {
        const uint32_t row = row_of(g), token = row >> a.group_shift, head = kv * a.group + (row & (a.group - 1));
        const V *qp = row_at<const V>(a.q, item.row0 + token, head);
        return *reinterpret_cast<const u32x4 *>(qp + (i >> 1) * 64 + quarter * 16 + (i & 1) * 8);
    };
#pragma unroll
    for (int g = 0; g < COLUMNS; g++) sees[g] = item.pos0 + int32_t(row_of(team * COLUMNS + g) >> a.group_shift) + 1;
    if constexpr (IN_LDS) {
#pragma unroll
        for (uint32_t i = wave; i < TILE_COLUMNS * 8; i += WAVES) q_lds[i / 8][i % 8][lane] = q_of(i / 8, i % 8);
    } else {
#pragma unroll
        for (int g = 0; g < COLUMNS; g++)
#pragma unroll
            for (int i = 0; i < 8; i++) q[g][i] = q_of(g, i);
    }
    auto query = [&](int g, int i) {
        if constexpr (IN_LDS) return q_lds[team * COLUMNS + g][i][lane];
        else return q[g][i];
    };
    if (steps) fetch(a.cache.values, 0, v);
    const float c = a.scale * 1.4426950408889634f;
    const uint32_t all_see = uint32_t(max(item.pos0 + 1, 0));  // of the first row, and so of all

    floatx4 acc[COLUMNS][16];
    float m[COLUMNS], l[COLUMNS];
#pragma unroll
    for (int g = 0; g < COLUMNS; g++) {
        m[g] = NO_MAXIMUM, l[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; i++) acc[g][i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    __syncthreads();  // nan_from is clear, the queries are in LDS

    while (steps) {
        const uint32_t here = min(steps, FEW_STEPS);
        for (uint32_t step = 0; step < here; step++) {
            const uint32_t key = (first + step * (2 * TURNS)) * UNIT_TOKENS;
            floatx4 s[COLUMNS][2];
#pragma unroll
            for (int g = 0; g < COLUMNS; g++) s[g][0] = s[g][1] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const u32x4 low = operands_of<TYPE>(k[i][j].x, k[i][j].y), high = operands_of<TYPE>(k[i][j].z, k[i][j].w);
#pragma unroll
                    for (int g = 0; g < COLUMNS; g++) s[g][i] = product16<TYPE>(low, query(g, 2 * j), s[g][i]);
#pragma unroll
                    for (int g = 0; g < COLUMNS; g++) s[g][i] = product16<TYPE>(high, query(g, 2 * j + 1), s[g][i]);
                }
            }
            if (step + 1 < here) fetch(a.cache.keys, step + 1, k);
            const uint32_t scale[2] = {uint32_t(__builtin_amdgcn_readlane(scales, 2 * step)), uint32_t(__builtin_amdgcn_readlane(scales, 2 * step + 1))};
            const ValueExponent exponents[2] = {value_exponent(scale[0]), value_exponent(scale[1])};
            const int ev[2] = {exponents[0].rest, exponents[1].rest};
            const float ck[2] = {c * key_scale(scale[0]), c * key_scale(scale[1])}, held[2] = {power_of_two(exponents[0].held), power_of_two(exponents[1].held)};
            const bool masked = key + STEP_KEYS > min(all_see, item.key1) || !(scale[0] & scale[1] & 0x10000);
            // (what follows from the lane is worked out where it is used: kept over the loop it would be in registers that the sums want)
            uint32_t at = lane;
            if (masked) {
                asm volatile("" : "+v"(at));
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const uint32_t from = key + i * UNIT_TOKENS + (at >> 4) * 4, limit = scale[i] & 0x10000 ? item.key1 : 0;
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int t = 0; t < 4; t++) v[i][j][t] = clean_values(v[i][j][t], from, limit, all_see, (4 * j + t) * 16 + (at & 15), nan_from);
                }
            }
            u32x4 w[COLUMNS], below[BOTH_HALVES ? COLUMNS : 1];
#pragma unroll
            for (int g = 0; g < COLUMNS; g++) {
                if (masked) {
                    // keys of the step that the row sees, less the quarter's four; none of a unit that is not there
                    const int n = min(sees[g], int(item.key1)) - int(key + (at >> 4) * 4);
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const int seen = scale[i] & 0x10000 ? n - i * int(UNIT_TOKENS) : -1;
#pragma unroll
                        for (int r = 0; r < 4; r++) s[g][i][r] = r < seen ? s[g][i][r] : NO_SCORE;
                    }
                }
                // (the scale is a power of two times a positive number: a unit's largest score is that of its largest product)
                float top = NO_SCORE;
#pragma unroll
                for (int i = 0; i < 2; i++) top = fmaxf(top, fmaf(fmaxf(fmaxf(s[g][i][0], s[g][i][1]), fmaxf(s[g][i][2], s[g][i][3])), ck[i], float(ev[i])));
                top = across_rows<16, 64>(top, MaxOp());
                if (__any(top > m[g] + (TOP + TAU))) {
                    const float next = top > m[g] + (TOP + TAU) ? top - TOP : m[g], down = __builtin_amdgcn_exp2f(m[g] - next);
                    m[g] = next, l[g] *= down;
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[g][i] *= down;
                }
                float p[2][4], part[2] = {0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 2; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) p[i][r] = __builtin_amdgcn_exp2f(fmaf(s[g][i][r], ck[i], float(ev[i]) - m[g])), part[i] += p[i][r];
                l[g] = fmaf(part[0], power_of_two(-ev[0]), fmaf(part[1], power_of_two(-ev[1]), l[g]));
                w[g] = u32x4{pack_half2(p[0][0], p[0][1]), pack_half2(p[0][2], p[0][3]), pack_half2(p[1][0], p[1][1]), pack_half2(p[1][2], p[1][3])};
                if constexpr (BOTH_HALVES) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t both = w[g][i];
                        const half2_ high = __builtin_bit_cast(half2_, both);
                        below[g][i] = pack_half2(p[i >> 1][i % 2 * 2] - float(high.x), p[i >> 1][i % 2 * 2 + 1] - float(high.y));
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int t = 0; t < 4; t++) {
                    const u32x2 v0 = halves_of(v[0][j][t], held[0]), v1 = halves_of(v[1][j][t], held[1]);
#pragma unroll
                    for (int g = 0; g < COLUMNS; g++) acc[g][4 * j + t] = product16<SAETTA_F16>(u32x4{v0.x, v0.y, v1.x, v1.y}, w[g], acc[g][4 * j + t]);
                    if constexpr (BOTH_HALVES) {
#pragma unroll
                        for (int g = 0; g < COLUMNS; g++) acc[g][4 * j + t] = product16<SAETTA_F16>(u32x4{v0.x, v0.y, v1.x, v1.y}, below[g], acc[g][4 * j + t]);
                    }
                }
            if (step + 1 < here) fetch(a.cache.values, step + 1, v);
        }
        steps -= here;
        if (steps) {
            first += FEW_STEPS * 2 * TURNS;
            look_up();
            fetch(a.cache.keys, 0, k);
            look_up_scales();
            fetch(a.cache.values, 0, v);
        }
    }

#pragma unroll
    for (int g = 0; g < TILE_COLUMNS; g++) {
        if (g > 0) {
            if (g * FEW_ROWS >= rows) return;
            __syncthreads();  // the last group's sums have been read
        }
        if (team == uint32_t(g / COLUMNS)) {
            const float sum_all = across_rows<16, 64>(l[g % COLUMNS], SumOp());
#pragma unroll
            for (int i = 0; i < 16; i++) *reinterpret_cast<floatx4 *>(&sums[turn][col][i * 16 + quarter * 4]) = acc[g % COLUMNS][i];
            if (quarter == 0) ml[turn][col][0] = m[g % COLUMNS], ml[turn][col][1] = sum_all;
        }
        __syncthreads();
        for (uint32_t i = wave; i < min(rows - g * FEW_ROWS, FEW_ROWS); i += WAVES) {
            const uint32_t r = g * FEW_ROWS + i, dim = lane * 4;
            float top = NO_MAXIMUM, sum = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < TURNS; w++) top = fmaxf(top, ml[w][i][0]);
#pragma unroll
            for (int w = 0; w < TURNS; w++) {
                const float f = __builtin_amdgcn_exp2f(ml[w][i][0] - top);
                sum = fmaf(ml[w][i][1], f, sum);
                const floatx4 x = *reinterpret_cast<const floatx4 *>(&sums[w][i][dim]);
#pragma unroll
                for (int d = 0; d < 4; d++) o[d] = fmaf(x[d], f, o[d]);
            }
            const uint32_t token = r >> a.group_shift;
#pragma unroll
            for (int d = 0; d < 4; d++)
                if (nan_from[dim + d] != ~0u && int32_t(nan_from[dim + d]) < item.pos0 + int32_t(token) + 1) o[d] = __builtin_nanf("");
            if (item.parts > 1) {
                const size_t slot = (size_t(item.slot) * a.cache.kv_heads + kv) * TILE + r;
                *reinterpret_cast<floatx4 *>(a.part_o + slot * DIM + dim) = floatx4{o[0], o[1], o[2], o[3]};
                if (lane == 0) *reinterpret_cast<float2 *>(a.part_ml + slot * 2) = float2{top, sum};
            } else {
                const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
                for (int d = 0; d < 4; d++) o[d] *= inv;
                put_row<TYPE>(a, item.row0 + token, kv * a.group + (r & (a.group - 1)), dim, o);
            }
        }
    }
}

template <int TYPE, int TILE_COLUMNS>
__global__ __launch_bounds__(few_threads(TILE_COLUMNS), TILE_COLUMNS == 2 ? 1 : 2) void paged_few_kernel(AttnArgs a) {
    constexpr int TEAMS = TILE_COLUMNS == 4 ? 2 : 1, COLUMNS = TILE_COLUMNS / TEAMS;
    __shared__ __attribute__((aligned(16))) FewShared<COLUMNS, TEAMS, FEW_WAVES> shared;
    __shared__ uint32_t nan_from[DIM];
    const uint32_t index = blockIdx.x / a.cache.kv_heads, kv = blockIdx.x % a.cache.kv_heads;
    const uint32_t items = a.head->items;
    const Item item = a.items[index];
    if (!(int(index < items) & int(item_ok(a, item, 1)))) return;
    take_few<TYPE, COLUMNS, TEAMS, FEW_WAVES, TILE_COLUMNS * FEW_ROWS>(a, item, kv, shared, nan_from);
}

// A workgroup barrier for what went through LDS: the copies of later steps stay on their way (__syncthreads waits for them).
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Chunks: a workgroup of 8 waves takes 256 rows (256 / group tokens of the q heads of a kv head), 32 a wave, over an item's keys, 32 a
// step.  The codes travel global -> LDS, AHEAD steps before they are wanted; the wave that asked for a kilobyte of keys and one of values
// makes halves of them, in the order of the operands, once for all eight waves.  A wave's step is a softmax and one stream of products, O^T +=
// V^T P^T of the step and S^T = K Q^T of the next; the two waves of a SIMD (w and w + 4) take them in opposite order, one's softmax and
// conversions under the other's products:
//   waves 0..3:  softmax(s)                | O(s) + S(s+1)
//   waves 4..7:  O(s) + S(s+1)             | softmax(s+1)
// Step s reads V(s) and K(s+1) as halves and makes V(s+1) and K(s+2), in the places of V(s-1) and K(s): one barrier a step.
// Bound by the matrix cores and the clock that they leave (1.8 GHz): 4096 tokens at 28672, bf16, 16 q heads over 2 kv heads, 1.75 to 1.93 ms, 1.07 to 1.18 PFLOP/s (a
// large product of the library on the same cards: 1.17 to 1.25); the streams of products alone 1.45 ms; without the priority that keeps the two waves in opposite order 2.28.  A short item
// is bound by its start and end, 13 to 16 us: seven prompts of 147 to 1645 tokens 73 us, a tile of 32 tokens 20.
constexpr uint32_t CODE_BYTES = STEP_KEYS * DIM, HALF_BYTES = 2 * CODE_BYTES;  // a step's keys, or values
constexpr uint32_t AHEAD = 3, PLACES = 4;
constexpr uint32_t K_HALVES = 0, V_HALVES = 2 * HALF_BYTES, K_CODES = 4 * HALF_BYTES, V_CODES = K_CODES + PLACES * CODE_BYTES;
constexpr uint32_t OUT_STRIDE = 128 + 4;  // floats of half a row on its way out, and the row's sum
constexpr uint32_t OUT_BYTES = CHUNK_ROWS * OUT_STRIDE * 4;
constexpr uint32_t TILE_LDS = OUT_BYTES > V_CODES + PLACES * CODE_BYTES ? OUT_BYTES : V_CODES + PLACES * CODE_BYTES;
constexpr uint32_t CHUNK_LDS = TILE_LDS > sizeof(FewShared<2, 1, CHUNK_WAVES>) ? TILE_LDS : sizeof(FewShared<2, 1, CHUNK_WAVES>);
template <int N>
struct Count {
    static constexpr int value = N;
};
template <int TYPE>
__global__ __launch_bounds__(64 * CHUNK_WAVES, 2) void paged_chunk_kernel(AttnArgs a) {
    typedef typename Row<TYPE>::value V;
    extern __shared__ __attribute__((aligned(1024))) unsigned char tiles[];
    __shared__ Unit units[WINDOW];
    __shared__ __attribute__((aligned(16))) uint32_t nan_from[DIM];
    constexpr bool BRAIN = TYPE == SAETTA_BF16;
    const uint32_t index = blockIdx.x / a.cache.kv_heads, kv = blockIdx.x % a.cache.kv_heads;
    const uint32_t items = a.head->items;
    const Item item = a.items[index];
    if (!(int(index < items) & int(item_ok(a, item, 1)))) return;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t rows = item.tokens << a.group_shift;
    // A draft beside a chunk, a prompt's last tokens.  (64 requests of 2, 4, 8 tokens at 4000, by this kernel: 46, 58, 73 us; by the one for few rows 46, 50, 68.
    // With one group to a wave and more teams, which spills no registers, 44, 70, 81.)
    if (rows <= 4 * FEW_ROWS) {
        auto few = [&](auto columns, auto teams) {
            constexpr int COLUMNS = decltype(columns)::value, TEAMS = decltype(teams)::value, TURNS = CHUNK_WAVES / TEAMS;
            typedef FewShared<COLUMNS, TEAMS, TURNS> Shared;
            static_assert(sizeof(Shared) <= CHUNK_LDS, "in the tiles' place");
            take_few<TYPE, COLUMNS, TEAMS, TURNS, CHUNK_ROWS>(a, item, kv, *reinterpret_cast<Shared *>(tiles), nan_from);
        };
        if (rows <= FEW_ROWS) few(Count<1>(), Count<1>());
        else if (rows <= 2 * FEW_ROWS) few(Count<2>(), Count<1>());
        else few(Count<2>(), Count<2>());
        return;
    }
    for (uint32_t i = tid; i < DIM; i += 64 * CHUNK_WAVES) nan_from[i] = ~0u;
    const uint32_t unit0 = item.key0 / UNIT_TOKENS, end_unit = (item.key1 + UNIT_TOKENS - 1) / UNIT_TOKENS;
    const uint32_t steps = end_unit > unit0 ? (end_unit - unit0 + 1) / 2 : 0;
    // What a wave holds of the units of 32 steps, unit j of step i in lane 2 i + j: where the codes to be copied are, and the scales of the steps that are
    // worked on.  (A lane's register is read at once; read from LDS each time, with nothing to do meanwhile, they were a third of a step.)  Those of
    // the first steps every wave looks up by itself: the queries' loads go out behind that one, and the codes' copies as soon as it is back.
    Unit unit = find_unit(a, item.request, kv, unit0 + lane, end_unit);
    uint32_t places = 0, scales = 0;

    half8 q[16];
    int32_t sees;
    {
        const uint32_t row = min(wave * 32 + (lane & 31), rows - 1), token = row >> a.group_shift, head = kv * a.group + (row & (a.group - 1));
        sees = item.pos0 + int32_t(token) + 1;
        const V *qp = row_at<const V>(a.q, item.row0 + token, head) + (lane >> 5) * 8;
#pragma unroll
        for (int i = 0; i < 16; i++) q[i] = *reinterpret_cast<const half8 *>(qp + i * 16);
    }
    const float c = a.scale * 1.4426950408889634f;
    const uint32_t all_see = uint32_t(max(item.pos0 + 1, 0));
    // what the wave's first and last rows see
    const uint32_t first_row = min(wave * 32, rows - 1), last_row = min(wave * 32 + 31, rows - 1);
    const uint32_t wave_all = min(uint32_t(max(item.pos0 + int32_t(first_row >> a.group_shift) + 1, 0)), item.key1);
    const uint32_t wave_end = wave * 32 < rows ? min(uint32_t(max(item.pos0 + int32_t(last_row >> a.group_shift) + 1, 0)), item.key1) : 0;

    floatx16 acc[8];
#pragma unroll
    for (int i = 0; i < 8; i++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][r] = 0.0f;
    float m = NO_MAXIMUM, l = 0.0f;

    const size_t block_bytes = size_t(DIM) << a.block_shift;
    const uint32_t unit_mask = (1u << (a.block_shift - 4)) - 1;
    const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>(tiles));
    // The lane, for what is worked out from it where it is used: kept over the loop it would be in registers that the queries want.
    auto here = [&] {
        uint32_t at = lane;
        asm volatile("" : "+v"(at));
        return at;
    };
    // the wave's kilobyte of a step: 64 dims (part) of the unit `mine`
    const uint32_t mine = wave >> 2, part = wave & 3;
    auto hold = [&](uint32_t step) { return units[(unit0 + 2 * step + here()) % WINDOW]; };
    auto copy = [&](const uint8_t *codes, uint32_t step, uint32_t place) {
        const uint32_t row = __builtin_amdgcn_readlane(places, (2 * step + mine) % 64);
        const uint64_t src = reinterpret_cast<uint64_t>(codes) + row * block_bytes + ((unit0 + 2 * step + mine) & unit_mask) * UNIT_BYTES + part * 1024;
        asm volatile(
            "s_mov_b32 m0, %[dst]\n"
            "s_nop 0\n"
            "global_load_lds_dwordx4 %[off], %[src]\n"
            :
            : [off] "v"(here() * 16), [src] "s"(src), [dst] "s"(lds0 + place + (step % PLACES) * CODE_BYTES + wave * 1024)
            : "memory", "m0");
    };
    auto copy_values = [&](uint32_t step) { copy(a.cache.values, step, V_CODES); };
    auto copy_keys = [&](uint32_t step) {  // (the keys are a step ahead of the values: the first to want the next 32)
        if (step % 32 == 0) places = step < steps ? hold(step).block : kv;  // (from the last step on: block 0, whose codes nobody looks at)
        copy(a.cache.keys, step, K_CODES);
    };
    auto keys_of = [&](uint32_t step) { return *reinterpret_cast<const u32x4 *>(tiles + K_CODES + (step % PLACES) * CODE_BYTES + wave * 1024 + here() * 16); };
    auto values_of = [&](uint32_t step) { return *reinterpret_cast<const u32x4 *>(tiles + V_CODES + (step % PLACES) * CODE_BYTES + wave * 1024 + here() * 16); };
    auto make_keys = [&](const u32x4 &x, uint32_t step) {  // token t, dims 64 part + 16 quarter .. + 15: both halves of fragment 4 part + quarter
        const uint32_t at = here(), t = at & 15, quarter = at >> 4;
        unsigned char *to = tiles + K_HALVES + (step & 1) * HALF_BYTES + (4 * part + quarter) * 1024 + (mine * 16 + t) * 16;
        *reinterpret_cast<u32x4 *>(to) = operands_of<TYPE>(x.x, x.y);
        *reinterpret_cast<u32x4 *>(to + 512) = operands_of<TYPE>(x.z, x.w);
    };
    auto make_values = [&](u32x4 x, uint32_t step) {  // tokens 4 quarter .. + 3 of dims 16 (4 part + i) + t
        const uint32_t at = here(), t = at & 15, quarter = at >> 4;
        const uint32_t key = (unit0 + 2 * step + mine) * UNIT_TOKENS;
        const uint32_t scale = __builtin_amdgcn_readlane(scales, (2 * step + mine) % 64);
        const bool there = scale & 0x10000;
        const float held = power_of_two(value_exponent(scale).held);
        if (key + UNIT_TOKENS > min(all_see, item.key1) || !there) {
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = clean_values(x[i], key + 4 * quarter, there ? item.key1 : 0, all_see, (4 * part + i) * 16 + t, nan_from);
        }
        unsigned char *to = tiles + V_HALVES + (step & 1) * HALF_BYTES + mine * 1024 + (quarter & 1) * 512 + (quarter >> 1) * 8;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t dim = (4 * part + i) * 16 + t;
            *reinterpret_cast<u32x2 *>(to + 2 * (dim >> 5) * 1024 + (dim & 31) * 16) = halves_of(x[i], held);
        }
    };
    // Probabilities of a step from its scores, as operands.
    auto softmax = [&](floatx16 &s, uint32_t step, half8 (&p)[2]) {
        const uint32_t key = (unit0 + 2 * step) * UNIT_TOKENS;
        const uint32_t scale[2] = {uint32_t(__builtin_amdgcn_readlane(scales, 2 * step % 64)), uint32_t(__builtin_amdgcn_readlane(scales, (2 * step + 1) % 64))};
        float ck[2], sum[2] = {0.0f, 0.0f}, tops[2] = {NO_SCORE, NO_SCORE};
        int ev[2];
#pragma unroll
        for (int i = 0; i < 2; i++) ck[i] = c * key_scale(scale[i]), ev[i] = value_exponent(scale[i]).rest;
        if (key + STEP_KEYS > wave_all || !(scale[0] & scale[1] & 0x10000)) {
            // keys of the step that the row sees, less the lane half's four; none of a unit that is not there
            const int n = min(sees, int(item.key1)) - int(key) - 4 * int(here() >> 5);
            const int seen[2] = {scale[0] & 0x10000 ? n : -1, scale[1] & 0x10000 ? n : -1};
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = int((r & 3) + 8 * (r >> 2)) < (r < 8 ? seen[0] : seen[1]) ? s[r] : NO_SCORE;
        }
        // (the scale is a power of two times a positive number: a unit's largest score is that of its largest product)
#pragma unroll
        for (int r = 0; r < 16; r++) tops[r >> 3] = fmaxf(tops[r >> 3], s[r]);
        const float top = across_rows<32, 64>(fmaxf(fmaf(tops[0], ck[0], float(ev[0])), fmaf(tops[1], ck[1], float(ev[1]))), MaxOp());
        if (__any(top > m + (TOP + TAU))) {
            const float next = top > m + (TOP + TAU) ? top - TOP : m, down = __builtin_amdgcn_exp2f(m - next);
            m = next, l *= down;
#pragma unroll
            for (int i = 0; i < 8; i++) acc[i] *= down;
        }
#pragma unroll
        for (int r = 0; r < 16; r++) s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], ck[r >> 3], float(ev[r >> 3]) - m)), sum[r >> 3] += s[r];
        l = fmaf(sum[0], power_of_two(-ev[0]), fmaf(sum[1], power_of_two(-ev[1]), l));
#pragma unroll
        for (int sp = 0; sp < 2; sp++) {
            const u32x4 w = {pack_half2(s[8 * sp], s[8 * sp + 1]), pack_half2(s[8 * sp + 2], s[8 * sp + 3]),
                             pack_half2(s[8 * sp + 4], s[8 * sp + 5]), pack_half2(s[8 * sp + 6], s[8 * sp + 7])};
            p[sp] = __builtin_bit_cast(half8, w);
        }
    };
    auto key_at = [&](uint32_t step) { return (unit0 + 2 * step) * UNIT_TOKENS; };
    auto k_halves = [&](uint32_t step) { return lds0 + K_HALVES + (step & 1) * HALF_BYTES + here() * 16; };
    auto v_halves = [&](uint32_t step) { return lds0 + V_HALVES + (step & 1) * HALF_BYTES + here() * 16; };

    if (steps) {
        // K(0), K(1), V(0), then what the steps before the first would have asked for
        places = unit.block;
        copy(a.cache.keys, 0, K_CODES), copy(a.cache.keys, 1, K_CODES), copy_values(0);
        scales = find_scales(a, unit);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_barrier();  // nan_from is clear
        make_keys(keys_of(0), 0), make_keys(keys_of(1), 1), make_values(values_of(0), 0);
        if (steps > 32 - (AHEAD + 2)) {  // the units of later steps: a window, from which a wave takes those of its next 32
            static_assert(WINDOW == 64 * CHUNK_WAVES, "a thread a unit");
            unit = find_unit(a, item.request, kv, unit0 + tid, end_unit);
            unit.scales = find_scales(a, unit);
            units[(unit0 + tid) % WINDOW] = unit;
        }
        static_assert(PLACES == AHEAD + 1, "a place is free again when the step after next asks for it");
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; i++) copy_values(1 + i), copy_keys(2 + i);
        lds_barrier();
        static_assert(AHEAD == 3, "the copies of three steps are on their way: six of a wave");
        auto begin = [&](uint32_t step) {
            // half of the window ahead, before a step comes near it
            if (step % (WINDOW / 4) == 0 && step && tid < WINDOW / 2) {
                const uint32_t u = unit0 + 2 * step + WINDOW / 2 + tid;
                unit = find_unit(a, item.request, kv, u, end_unit);
                unit.scales = find_scales(a, unit);
                units[u % WINDOW] = unit;
            }
            copy_values(step + 1 + AHEAD), copy_keys(step + 2 + AHEAD);
        };
        auto arrived = [&] { asm volatile("s_waitcnt vmcnt(6)" ::: "memory"); };  // V(step + 1), K(step + 2)
        if (wave < 4) {
            floatx16 s;
            if (key_at(0) < wave_end) scores_block<BRAIN>(s, q, k_halves(0));
            lds_barrier();  // K(0) has been read
            for (uint32_t step = 0; step < steps; step++) {
                begin(step);
                arrived();
                const u32x4 v_codes = values_of(step + 1), k_codes = keys_of(step + 2);
                half8 p[2];
                const bool works = key_at(step) < wave_end;
                if (works) softmax(s, step, p);
                if ((step + 1) % 32 == 0) scales = step + 1 < steps ? hold(step + 1).scales : 0;
                make_values(v_codes, step + 1), make_keys(k_codes, step + 2);
                if (works) stream_block_alone<BRAIN>(s, acc, q, p, k_halves(step + 1), v_halves(step));
                lds_barrier();
            }
        } else {
            half8 p[2] = {};
            if (key_at(0) < wave_end) {
                floatx16 s;
                scores_block<BRAIN>(s, q, k_halves(0));
                softmax(s, 0, p);
            }
            lds_barrier();
            for (uint32_t step = 0; step < steps; step++) {
                begin(step);
                floatx16 s;
                const bool works = key_at(step) < wave_end;
                if (works) {
                    // (its products go first: its softmax then finds the other wave's to run under)
                    __builtin_amdgcn_s_setprio(2);
                    stream_block_alone<BRAIN>(s, acc, q, p, k_halves(step + 1), v_halves(step));
                    __builtin_amdgcn_s_setprio(0);
                }
                arrived();
                const u32x4 v_codes = values_of(step + 1), k_codes = keys_of(step + 2);
                if ((step + 1) % 32 == 0) scales = step + 1 < steps ? hold(step + 1).scales : 0;
                if (works && key_at(step + 1) < wave_end) softmax(s, step + 1, p);
                make_values(v_codes, step + 1), make_keys(k_codes, step + 2);
                lds_barrier();
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        settle(acc);
    }

    const uint32_t at = here();
    const uint32_t wave_rows = wave * 32 < rows ? min(rows - wave * 32, 32u) : 0, head0 = kv * a.group, in_half = 4 * (at & 31);
    auto in_wave = [&](int i) { return 2 * i + (at >> 5); };
    // Rows 2 i and 2 i + 1 are a head apart, or, of one head, a token: a lane's part of the address is the same for all i
    auto place_of = [&](int i, const Rows &rows_of) {
        const uint32_t row = wave * 32 + 2 * i;
        return row_at<V>(rows_of, item.row0 + (row >> a.group_shift), head0 + (row & (a.group - 1))) + (uint64_t((at >> 5) * (a.group > 1 ? rows_of.head_stride : rows_of.token_stride)) + in_half);
    };
    // (the gates of a half of the dims travel while what comes before them is done)
    const bool gated = a.gate.data && item.parts == 1;
    typedef V value4 __attribute__((ext_vector_type(4)));
    value4 gates[2][16];
    auto get_gates = [&](int half) {
        if (!gated) return;
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (in_wave(i) < wave_rows) gates[half][i] = *reinterpret_cast<const value4 *>(place_of(i, a.gate) + 128 * half);
    };
    get_gates(0);
    lds_barrier();  // nan_from is whole, and what the tiles held has been read
    // Through LDS, a half of the dims at a time, so that a wave stores two rows' 128 dims side by side.  A row's sum is behind its dims.
    l = across_rows<32, 64>(l, SumOp());
    float *mine_out = reinterpret_cast<float *>(tiles) + wave * (32 * OUT_STRIDE);
    mine_out[(at & 31) * OUT_STRIDE + 128] = l == 0.0f ? 0.0f : 1.0f / l;
    if (wave_rows == 0) return;
    if (item.parts > 1 && at < wave_rows)
        *reinterpret_cast<float2 *>(a.part_ml + ((size_t(item.slot) * a.cache.kv_heads + kv) * CHUNK_ROWS + wave * 32 + at) * 2) = float2{m, l};
#pragma unroll
    for (int half = 0; half < 2; half++) {
        wave_sync();  // the last half has been read
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const floatx16 &x = acc[4 * half + i];
                *reinterpret_cast<floatx4 *>(mine_out + (at & 31) * OUT_STRIDE + 32 * i + 4 * (at >> 5) + 8 * k) = floatx4{x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]};
            }
        if (half == 0) get_gates(1);
        const uint32_t dim = 128 * half + in_half;
        const uint4 nan4 = *reinterpret_cast<const uint4 *>(nan_from + dim);
        const uint32_t nans[4] = {nan4.x, nan4.y, nan4.z, nan4.w};
        const bool any_nan = (nans[0] & nans[1] & nans[2] & nans[3]) != ~0u;
        wave_sync();
        // (what is read is asked for eight rows at a time, with no branch but the stores' between: row by row the reads' latencies were 6 us of
        // a tile's end)
#pragma unroll
        for (int i0 = 0; i0 < 16; i0 += 8) {
            floatx4 o[8];
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = *reinterpret_cast<const floatx4 *>(mine_out + in_wave(i0 + i) * OUT_STRIDE + in_half);
            if (any_nan) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int32_t row_sees = item.pos0 + int32_t((wave * 32 + in_wave(i0 + i)) >> a.group_shift) + 1;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (nans[j] != ~0u && int32_t(nans[j]) < row_sees) o[i][j] = __builtin_nanf("");
                }
            }
            if (item.parts > 1) {
                float *part = a.part_o + ((size_t(item.slot) * a.cache.kv_heads + kv) * CHUNK_ROWS + wave * 32) * DIM + dim;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (uint32_t(in_wave(i0 + i)) < wave_rows) *reinterpret_cast<floatx4 *>(part + in_wave(i0 + i) * DIM) = o[i];
                continue;
            }
            float inv[8];
#pragma unroll
            for (int i = 0; i < 8; i++) inv[i] = mine_out[in_wave(i0 + i) * OUT_STRIDE + 128];
            value4 w[8];
            if (gated) {
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) w[i][j] = Row<TYPE>::store(o[i][j] * inv[i] * sigmoid(Row<TYPE>::load(gates[half][i0 + i][j])));
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) w[i][j] = Row<TYPE>::store(o[i][j] * inv[i]);
            }
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (uint32_t(in_wave(i0 + i)) < wave_rows) *reinterpret_cast<value4 *>(place_of(i0 + i, a.out) + 128 * half) = w[i];
        }
    }
}

// Joins the parts of the tiles that were taken in parts: out = sum_p 2^(M_p - M) O_p / sum_p 2^(M_p - M) l_p.  A lane has four dims of a row.  WIDE:
// a workgroup a row, the parts dealt to its four waves in turn; 3 to 5 us of few rows, by latency: the tile, then maxima, sums, parts and gate at once,
// then the output.  Of chunks, whose parts are 256 KB an item and kv head, up to WIDE_TILES tiles are joined so too; else a wave takes two rows, one
// after the other, for an eighth of the workgroups to launch: 11 to 17 us.
// (Joining in the attention kernel, by the workgroup that ends last, costs more than this launch: all workgroups run at once, so their stores' way
// to the memory that the XCDs share, the count and the loads come on top of the longest walk; 48 ragged contexts 67 -> 72 us, one of 517 tokens 9.3
// -> 9.7.)
constexpr uint32_t MERGE_ROWS = 2;  // seven prompts 13.2 us with 1, 10.9 with 2, 11.9 with 4; a chunk at 28672 16.8, 13.0, 13.4
// 32 tokens at 8000 (2 tiles at most) 17.1 us by waves, 10.9 wide; 100 at 3000 (4) 9.5 and 7.2; 200 at 20000 (7) 12.1 and 12.6; 300 at 0 (10) 4.6 and 5.9; seven
// prompts 10.9 and 31.9.
constexpr uint32_t WIDE_TILES = 6;
template <int TYPE, uint32_t TILE, bool WIDE>
__global__ __launch_bounds__(256) void paged_merge_kernel(AttnArgs a, const Item *tiles) {
    typedef typename Row<TYPE>::value V;
    constexpr uint32_t BY = WIDE ? 4 : 1, AT_ONCE = WIDE ? 8 : 4;
    const uint32_t there = a.head->tiles, kv = blockIdx.z;
    const Item item = tiles[blockIdx.x];
    if (!(int(blockIdx.x < there) & int(item.parts > 1) & int(item_ok(a, item, item.parts)))) return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rows = item.tokens << a.group_shift, r0 = WIDE ? blockIdx.y : (blockIdx.y * 4 + wave) * MERGE_ROWS;
    if (WIDE && r0 >= rows) return;  // (the whole workgroup)
    for (uint32_t r = r0; r < (WIDE ? r0 + 1 : min(r0 + MERGE_ROWS, rows)); r++) {
        const size_t stride = size_t(a.cache.kv_heads) * TILE, slot = (size_t(item.slot) * a.cache.kv_heads + kv) * TILE + r;
        const uint32_t row = item.row0 + (r >> a.group_shift);
        const uint32_t head = kv * a.group + (r & (a.group - 1)), dim = lane * 4;
        float gate[4];
        if (a.gate.data) load_values<TYPE, 4>(row_at<const V>(a.gate, row, head) + dim, gate);

        float m = NO_MAXIMUM, l = 0.0f;
        floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t p0 = WIDE ? wave : 0; p0 < item.parts; p0 += BY * AT_ONCE) {
            float2 ml[AT_ONCE];
            floatx4 x[AT_ONCE];
#pragma unroll
            for (uint32_t i = 0; i < AT_ONCE; i++) {
                ml[i] = float2{NO_MAXIMUM, 0.0f}, x[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
                if (p0 + i * BY < item.parts) {  // (for the wave alike)
                    const size_t at = slot + (p0 + i * BY) * stride;
                    ml[i] = *reinterpret_cast<const float2 *>(a.part_ml + at * 2);
                    x[i] = *reinterpret_cast<const floatx4 *>(a.part_o + at * DIM + dim);
                }
            }
            float top = m;
#pragma unroll
            for (uint32_t i = 0; i < AT_ONCE; i++) top = fmaxf(top, ml[i].x);
            const float down = __builtin_amdgcn_exp2f(m - top);
            m = top, l *= down, o *= down;
#pragma unroll
            for (uint32_t i = 0; i < AT_ONCE; i++) {
                const float f = __builtin_amdgcn_exp2f(ml[i].x - top);
                l = fmaf(ml[i].y, f, l);
#pragma unroll
                for (int j = 0; j < 4; j++) o[j] = fmaf(x[i][j], f, o[j]);
            }
        }
        if constexpr (WIDE) {
            __shared__ __attribute__((aligned(16))) float part[4][64][4];
            __shared__ float pml[4][2];
            *reinterpret_cast<floatx4 *>(part[wave][lane]) = o;
            if (lane == 0) pml[wave][0] = m, pml[wave][1] = l;
            __syncthreads();
            if (wave > 0) return;
            float top = NO_MAXIMUM;
#pragma unroll
            for (int w = 0; w < 4; w++) top = fmaxf(top, pml[w][0]);
            l = 0.0f, o = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = __builtin_amdgcn_exp2f(pml[w][0] - top);
                l = fmaf(pml[w][1], f, l);
                const floatx4 x = *reinterpret_cast<const floatx4 *>(part[w][lane]);
#pragma unroll
                for (int i = 0; i < 4; i++) o[i] = fmaf(x[i], f, o[i]);
            }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = a.gate.data ? o[i] * inv * sigmoid(gate[i]) : o[i] * inv;
        store_values<TYPE, 4>(row_at<V>(a.out, row, head) + dim, x);
    }
}

int check_attn(const saetta_paged_attn_params &p, uint32_t requests, const char *what) {
    SAETTA_REQUIRE(p.kv_heads > 0 && p.heads % p.kv_heads == 0 && p.kv_heads <= 32767, SAETTA_E_SHAPE, "%s: %u q heads over %u kv heads", what, p.heads, p.kv_heads);
    const uint32_t group = p.heads / p.kv_heads;
    SAETTA_REQUIRE(group == 1 || group == 2 || group == 4 || group == 8 || group == 16, SAETTA_E_SHAPE, "%s: %u q heads per kv head (1, 2, 4, 8 or 16)", what, group);
    SAETTA_REQUIRE(p.tokens < (1u << 31) && requests < (1u << 24), SAETTA_E_SHAPE, "%s: %u tokens of %u requests", what, p.tokens, requests);
    SAETTA_REQUIRE(p.rows > 0, SAETTA_E_SHAPE, "%s: rows 0", what);
    // (the largest score is taken from the largest product)
    SAETTA_REQUIRE(p.scale >= 0x1p-60f && p.scale <= 0x1p60f, SAETTA_E_SHAPE, "%s: scale %g (2^-60 to 2^60)", what, double(p.scale));
    // (one workgroup of up to 512 threads to an item and kv head: fewer than 2^32 threads)
    SAETTA_REQUIRE(uint64_t(shape_of(p, requests).most_items) * p.kv_heads < (1u << 23), SAETTA_E_SHAPE, "%s: %u tokens of %u requests over %u kv heads", what,
                   p.tokens, requests, p.kv_heads);
    return SAETTA_OK;
}
int check_batch(const saetta_paged_batch &b, const char *what) {
    SAETTA_REQUIRE(b.query_starts && b.kv_lens && b.block_table, SAETTA_E_NULL, "%s: null buffer", what);
    SAETTA_REQUIRE(aligned(b.query_starts, 4) && aligned(b.kv_lens, 4) && aligned(b.block_table, 4), SAETTA_E_ALIGN, "%s: the batch must be 4-byte aligned", what);
    SAETTA_REQUIRE(block_tokens_ok(b.block_tokens), SAETTA_E_SHAPE, "%s: blocks of %u tokens (16, 32, 64 or 128)", what, b.block_tokens);
    SAETTA_REQUIRE(b.max_blocks > 0 && uint64_t(b.max_blocks) * b.block_tokens < (1ull << 31), SAETTA_E_SHAPE, "%s: rows of %u blocks", what, b.max_blocks);
    return SAETTA_OK;
}
size_t items_offset() { return sizeof(SplitHead); }
size_t tiles_offset(const Shape &s) { return items_offset() + sizeof(Item) * s.most_items; }

// Whether no two of the rows overlap.  (Strides from 0 up: rows h heads and t tokens apart, and the same with h taken back, are |h head_stride - t token_stride| apart
// at least; of a head's t the two next to its place are the nearest.)
bool rows_apart(const saetta_strided_rows &r, uint64_t tokens, uint64_t heads) {
    const uint64_t ts = r.token_stride, hs = r.head_stride;
    if ((heads == 1 || hs >= DIM) && (tokens <= 1 || ts >= (heads - 1) * hs + DIM)) return true;
    for (uint64_t h = 0; h < heads; h++) {
        const uint64_t at = h * hs, t0 = ts ? at / ts : 0;
        for (uint64_t t = t0; t <= t0 + 1; t++)
            if (t < tokens && (h || t) && (at > t * ts ? at - t * ts : t * ts - at) < DIM) return false;
    }
    return true;
}
Rows narrow(const saetta_strided_rows &r) { return {r.data, uint32_t(r.token_stride), uint32_t(r.head_stride)}; }
uint32_t shift_of(uint32_t n) { return uint32_t(__builtin_ctz(n)); }

template <int TYPE>
void launch_attn(hipStream_t stream, const AttnArgs &a, const Shape &s, const saetta_paged_attn_params &p, const Item *tiles) {
    const dim3 grid(s.most_items * p.kv_heads);
    auto merge_wide = [&](auto merge) { launch(merge, dim3(s.most_joined, s.columns ? p.rows * s.group : CHUNK_ROWS, p.kv_heads), dim3(256), 0, stream, a, tiles); };
    auto few = [&](auto attention, auto merge) {
        launch(attention, grid, dim3(few_threads(int(s.columns))), 0, stream, a);
        merge_wide(merge);
    };
    switch (s.columns) {
        case 1: return few(paged_few_kernel<TYPE, 1>, paged_merge_kernel<TYPE, FEW_ROWS, true>);
        case 2: return few(paged_few_kernel<TYPE, 2>, paged_merge_kernel<TYPE, 2 * FEW_ROWS, true>);
        case 4: return few(paged_few_kernel<TYPE, 4>, paged_merge_kernel<TYPE, 4 * FEW_ROWS, true>);
    }
    launch(paged_chunk_kernel<TYPE>, grid, dim3(64 * CHUNK_WAVES), CHUNK_LDS, stream, a);
    if (s.most_joined <= WIDE_TILES) merge_wide(paged_merge_kernel<TYPE, CHUNK_ROWS, true>);
    else launch(paged_merge_kernel<TYPE, CHUNK_ROWS, false>, dim3(s.most_joined, CHUNK_ROWS / 4 / MERGE_ROWS, p.kv_heads), dim3(256), 0, stream, a, tiles);
}

}  // namespace

int setup_paged_attn() {
    for (const void *k : {reinterpret_cast<const void *>(paged_chunk_kernel<SAETTA_F16>), reinterpret_cast<const void *>(paged_chunk_kernel<SAETTA_BF16>)}) {
        if (int rc = load_kernel(k)) return rc;
        if (int rc = int(hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize, CHUNK_LDS))) return rc;
    }
    return 0;
}

}  // namespace saetta

using namespace saetta;

extern "C" size_t saetta_paged_split_bytes(saetta_paged_attn_params p, uint32_t requests) {
    if (check_attn(p, requests, "paged_split_bytes")) return 0;
    const Shape s = shape_of(p, requests);
    return tiles_offset(s) + sizeof(Item) * size_t(s.most_joined);
}

extern "C" size_t saetta_paged_workspace_bytes(saetta_paged_attn_params p, uint32_t requests) {
    if (check_attn(p, requests, "paged_workspace_bytes")) return 0;
    const Shape s = shape_of(p, requests);
    return size_t(s.slots) * p.kv_heads * s.tile_rows * (DIM + 2) * sizeof(float);
}

extern "C" int saetta_paged_split(saetta_stream_t stream, saetta_paged_batch batch, saetta_paged_attn_params p, void *split) {
    if (int rc = check_attn(p, batch.requests, "paged_split")) return rc;
    if (int rc = check_batch(batch, "paged_split")) return rc;
    SAETTA_REQUIRE(split, SAETTA_E_NULL, "paged_split: null buffer");
    SAETTA_REQUIRE(aligned(split, 16), SAETTA_E_ALIGN, "paged_split: split must be 16-byte aligned");
    if (int rc = ensure_device()) return rc;
    const Shape s = shape_of(p, batch.requests);
    unsigned char *at = static_cast<unsigned char *>(split);
    const bool few = s.columns > 0;
    const SplitArgs a = {batch, reinterpret_cast<SplitHead *>(at), reinterpret_cast<Item *>(at + items_offset()), reinterpret_cast<Item *>(at + tiles_offset(s)),
                         s.tile_tokens, s.target, s.most_items, s.most_joined, s.slots, p.tokens, p.rows,
                         few, few ? STEP_KEYS * FEW_WAVES : STEP_KEYS, LEAST_KEYS, few ? 0u : CHUNK_EXTRA, few ? 0u : 4 * FEW_ROWS / s.group, few ? 0u : s.tile_tokens / 2};
    // (few tiles: four waves, whose barriers are cheaper)
    if (s.most_tiles <= 256) launch(paged_split_kernel<256>, dim3(1), dim3(256), 0, as_stream(stream), a);
    else launch(paged_split_kernel<1024>, dim3(1), dim3(1024), 0, as_stream(stream), a);
    return launch_status("paged_split");
}

extern "C" int saetta_paged_attn(saetta_stream_t stream, int type, saetta_strided_rows q, saetta_paged_cache cache, saetta_paged_batch batch,
                                 const void *split, saetta_strided_rows gate, saetta_strided_rows out, saetta_paged_attn_params p, void *workspace,
                                 size_t workspace_bytes) {
    SAETTA_REQUIRE(type == SAETTA_F16 || type == SAETTA_BF16, SAETTA_E_BITS, "paged_attn: type %d (f16 or bf16)", type);
    if (int rc = check_attn(p, batch.requests, "paged_attn")) return rc;
    if (int rc = check_batch(batch, "paged_attn")) return rc;
    if (int rc = check_cache(cache, "paged_attn")) return rc;
    SAETTA_REQUIRE(cache.kv_heads == p.kv_heads && cache.block_tokens == batch.block_tokens, SAETTA_E_SHAPE,
                   "paged_attn: a cache of %u kv heads and blocks of %u tokens, a call of %u and %u", cache.kv_heads, cache.block_tokens, p.kv_heads, batch.block_tokens);
    SAETTA_REQUIRE(q.data && out.data && split && workspace, SAETTA_E_NULL, "paged_attn: null buffer");
    SAETTA_REQUIRE(rows_aligned(q, type) && rows_aligned(out, type) && rows_aligned(gate, type), SAETTA_E_ALIGN,
                   "paged_attn: q, gate and out must be 16-byte aligned, with strides of multiples of 16 bytes");
    for (const saetta_strided_rows &r : {q, gate, out})
        SAETTA_REQUIRE(r.token_stride < (1ull << 32) && r.head_stride < (1ull << 32), SAETTA_E_SHAPE, "paged_attn: strides of %llu and %llu values (less than 2^32)",
                       static_cast<unsigned long long>(r.token_stride), static_cast<unsigned long long>(r.head_stride));
    SAETTA_REQUIRE(rows_apart(out, p.tokens, p.heads), SAETTA_E_SHAPE, "paged_attn: out's rows overlap (strides of %llu and %llu values)",
                   static_cast<unsigned long long>(out.token_stride), static_cast<unsigned long long>(out.head_stride));
    SAETTA_REQUIRE(aligned(split, 16) && aligned(workspace, 16), SAETTA_E_ALIGN, "paged_attn: split and workspace must be 16-byte aligned");
    const size_t need = saetta_paged_workspace_bytes(p, batch.requests);
    SAETTA_REQUIRE(workspace_bytes >= need, SAETTA_E_SCRATCH, "paged_attn: workspace of %zu bytes (%zu needed)", workspace_bytes, need);
    if (int rc = ensure_device()) return rc;
    if (batch.requests == 0 || p.tokens == 0) return SAETTA_OK;
    const Shape s = shape_of(p, batch.requests);
    const unsigned char *at = static_cast<const unsigned char *>(split);
    float *part_o = static_cast<float *>(workspace);
    const AttnArgs a = {narrow(q), narrow(gate), narrow(out), cache, batch.block_table, reinterpret_cast<const SplitHead *>(at), reinterpret_cast<const Item *>(at + items_offset()),
                        part_o, part_o + size_t(s.slots) * p.kv_heads * s.tile_rows * DIM, batch.requests, batch.max_blocks, p.tokens,
                        s.group, shift_of(s.group), shift_of(cache.block_tokens), s.slots, s.tile_tokens, p.scale};
    const Item *tiles = reinterpret_cast<const Item *>(at + tiles_offset(s));
    if (type == SAETTA_F16) launch_attn<SAETTA_F16>(as_stream(stream), a, s, p, tiles);
    else launch_attn<SAETTA_BF16>(as_stream(stream), a, s, p, tiles);
    return launch_status("paged_attn");
}
