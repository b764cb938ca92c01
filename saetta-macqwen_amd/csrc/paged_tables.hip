// Block tables, slots and positions of a step, from the lengths of the requests.
//
// want[r] = min(ceil((context[r] + new[r]) / block), max_blocks).  A request that holds fewer takes what is missing out of
// one segment at the end of the free list, request by request (an exclusive prefix sum of what they take); one that holds
// more gives the rest back behind what is left of the list, in the same order (another prefix sum).  So what a step takes
// and the next gives back whole leaves the list as it was.  The tokens' first rows are a third prefix sum.
//
// Bound by latency: a few bytes a request, two numbers a token.  The sums want every request, so one workgroup of 1024
// makes them, requests 1024 at a time, and moves the blocks' numbers, entry by entry over all its threads (a request is
// found by bisection in the prefix sums in LDS).  The tokens' slots are independent of each other: a second launch of as
// many workgroups as they fill, or, where few workgroups' worth of tokens come (a decode step), the first does them itself.
#include "common.hpp"
#include "lanes.hpp"
#include "paged_device.hpp"

namespace saetta {
namespace {

constexpr int TABLE_THREADS = 1024, TABLE_WAVES = TABLE_THREADS / 64;
constexpr uint32_t SLOT_TOKENS = 1024;  // of a workgroup of the second launch

struct TablesArgs {
    const uint32_t *context_lens, *new_lens;
    saetta_paged_state state;
    saetta_paged_step step;
    saetta_paged_tables_params p;
};

// Sums stop at the largest number there is (every order of adding gives the same).
__device__ __forceinline__ uint32_t add_up(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }

// x summed over the threads before this one; `all`: over all of them.  (All threads; `waves` is free again on return.)
__device__ __forceinline__ uint32_t sum_before(uint32_t x, uint32_t *waves, uint32_t &all) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t through = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t other = __shfl_up(through, d);
        if (lane >= uint32_t(d)) through = add_up(through, other);
    }
    if (lane == 63) waves[wave] = through;
    __syncthreads();
    uint32_t before = 0;
    all = 0;
#pragma unroll
    for (uint32_t w = 0; w < TABLE_WAVES; w++) {
        if (w == wave) before = all;
        all = add_up(all, waves[w]);
    }
    __syncthreads();
    const uint32_t prior = __shfl_up(through, 1);
    return add_up(before, lane == 0 ? 0 : prior);
}

struct Lengths {
    uint32_t context, fresh, held, want;
};
__device__ __forceinline__ Lengths lengths_of(const TablesArgs &a, uint32_t r) {
    Lengths l = {0, 0, 0, 0};
    if (r < a.p.requests) {
        l.context = a.context_lens[r], l.fresh = a.new_lens[r], l.held = min(a.state.held[r], a.p.max_blocks);
        const uint32_t length = add_up(l.context, l.fresh), bt = a.p.block_tokens;
        l.want = min(length / bt + (length % bt != 0), a.p.max_blocks);
    }
    return l;
}

// The last of `starts` (rising, starts[0] <= x) that is no more than x.
template <class T>
__device__ __forceinline__ uint32_t last_at_most(const T *starts, uint32_t n, uint32_t x) {
    uint32_t low = 0;
    while (n > 1) {
        const uint32_t half = n / 2;
        if (starts[low + half] <= x) low += half, n -= half;
        else n = half;
    }
    return low;
}

// Token t's slot and position (-1 past the step's last token).  Whether it has a slot.
__device__ __forceinline__ bool place_token(const TablesArgs &a, uint32_t t, uint32_t total) {
    int32_t slot = -1, position = -1;
    if (t < total) {
        // (requests without new tokens share their start with the next: the last of them is the token's)
        const uint32_t r = last_at_most(a.step.query_starts, a.p.requests, t), bt = a.p.block_tokens;
        // (from the sum and not from context_lens, which kv_lens may be: those have grown by now)
        const uint32_t context = a.step.kv_lens[r] - a.new_lens[r], at = add_up(context, t - a.step.query_starts[r]);
        position = int32_t(min(at, 0x7fffffffu));
        const uint32_t entry = at / bt;
        if (entry < min(a.state.held[r], a.p.max_blocks)) {
            const uint32_t block = uint32_t(a.state.block_table[size_t(r) * a.p.max_blocks + entry]);
            if (block < a.p.blocks) slot = int32_t(block * bt + at % bt);
        }
    }
    a.step.slots[t] = slot, a.step.positions[t] = position;
    return slot >= 0;
}

template <bool SLOTS>
__global__ __launch_bounds__(TABLE_THREADS) void paged_tables_kernel(TablesArgs a) {
    __shared__ uint32_t waves[TABLE_WAVES], starts[TABLE_THREADS], firsts[TABLE_THREADS];
    const uint32_t tid = threadIdx.x, requests = a.p.requests, room = a.p.tokens;
    const uint32_t free_count = min(*a.state.free_count, a.p.blocks);

    // what is taken and given in all, and the step's tokens
    uint32_t takes = 0, gives = 0, total = 0;
    for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
        const Lengths l = lengths_of(a, r0 + tid);
        takes = add_up(takes, l.want > l.held ? l.want - l.held : 0);
        gives = add_up(gives, l.held > l.want ? l.held - l.want : 0);
        total = add_up(total, l.fresh);
    }
    uint32_t all_takes, all_gives, all_tokens;
    sum_before(takes, waves, all_takes), sum_before(gives, waves, all_gives), sum_before(total, waves, all_tokens);
    const uint32_t taken = min(all_takes, free_count), left = free_count - taken;
    total = min(all_tokens, room);

    // blocks that are taken; the requests' first tokens and lengths
    uint32_t takes_before = 0, tokens_before = 0;
    for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
        const uint32_t r = r0 + tid;
        const Lengths l = lengths_of(a, r);
        const uint32_t take = l.want > l.held ? l.want - l.held : 0;
        uint32_t here;
        const uint32_t token = add_up(tokens_before, sum_before(l.fresh, waves, here));
        tokens_before = add_up(tokens_before, here);
        const uint32_t before = add_up(takes_before, sum_before(take, waves, here));
        takes_before = add_up(takes_before, here);
        if (r < requests) {
            a.step.query_starts[r] = min(token, room);
            a.step.kv_lens[r] = add_up(l.context, l.fresh);
            if (take > 0) a.state.held[r] = l.held + min(take, taken - min(before, taken));
        }
        if (here == 0) continue;  // (for all threads alike)
        starts[tid] = before, firsts[tid] = l.held;
        __syncthreads();
        const uint32_t first = starts[0], end = min(takes_before, taken), n = min(TABLE_THREADS, int(requests - r0));
        for (uint32_t k = first + tid; k < end; k += TABLE_THREADS) {
            const uint32_t i = last_at_most(starts, n, k);
            a.state.block_table[size_t(r0 + i) * a.p.max_blocks + firsts[i] + (k - starts[i])] = a.state.free_list[left + k];
        }
        __syncthreads();
    }
    if (tid == 0) {
        a.step.query_starts[requests] = total;
        *a.state.free_count = min(add_up(left, all_gives), a.p.blocks);
    }
    __syncthreads();  // what is taken has been read: what is given may land there

    if (all_gives > 0) {
        uint32_t gives_before = 0;
        for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
            const uint32_t r = r0 + tid;
            // (lengths from kv_lens: context_lens may be the same array)
            Lengths l = {0, 0, 0, 0};
            if (r < requests) {
                l.held = min(a.state.held[r], a.p.max_blocks);
                const uint32_t length = a.step.kv_lens[r], bt = a.p.block_tokens;
                l.want = min(length / bt + (length % bt != 0), a.p.max_blocks);
            }
            const uint32_t give = l.held > l.want ? l.held - l.want : 0;
            uint32_t here;
            const uint32_t before = add_up(gives_before, sum_before(give, waves, here));
            gives_before = add_up(gives_before, here);
            if (here == 0) continue;
            starts[tid] = before, firsts[tid] = l.want;
            __syncthreads();
            const uint32_t first = starts[0], n = min(TABLE_THREADS, int(requests - r0));
            for (uint32_t k = first + tid; k < gives_before; k += TABLE_THREADS) {
                const uint32_t i = last_at_most(starts, n, k);
                int32_t *entry = a.state.block_table + size_t(r0 + i) * a.p.max_blocks + firsts[i] + (k - starts[i]);
                // (more than the list has room for: a table that names blocks twice; they are lost, not written past its end)
                if (left + k < a.p.blocks) a.state.free_list[left + k] = *entry;
                *entry = -1;
            }
            __syncthreads();
            if (give > 0) a.state.held[r] = l.want;
        }
    }

    if constexpr (SLOTS) {
        __syncthreads();
        uint32_t placed = 0;
        for (uint32_t t = tid; t < room; t += TABLE_THREADS) placed += place_token(a, t, total);
        uint32_t all;
        sum_before(placed, waves, all);
        if (tid == 0) *a.step.unplaced = all_tokens - all;
    } else {
        if (tid == 0) *a.step.unplaced = all_tokens;  // the second launch takes off what it places
    }
}

// The second launch: SLOT_TOKENS tokens a workgroup.
__global__ __launch_bounds__(256) void paged_slots_kernel(TablesArgs a) {
    const uint32_t total = a.step.query_starts[a.p.requests];
    uint32_t placed = 0;
#pragma unroll
    for (uint32_t i = 0; i < SLOT_TOKENS; i += 256) {
        const uint64_t t = uint64_t(blockIdx.x) * SLOT_TOKENS + i + threadIdx.x;
        const bool has = t < a.p.tokens && place_token(a, uint32_t(t), total);
        placed += __popcll(__ballot(has));
    }
    if ((threadIdx.x & 63) == 0 && placed > 0) atomicSub(a.step.unplaced, placed);  // (whole numbers: any order gives the same)
}

}  // namespace

int setup_paged_tables() { return load_kernel(reinterpret_cast<const void *>(paged_slots_kernel)); }

}  // namespace saetta

using namespace saetta;

extern "C" int saetta_paged_tables(saetta_stream_t stream, const uint32_t *context_lens, const uint32_t *new_lens,
                                   saetta_paged_state state, saetta_paged_step step, saetta_paged_tables_params p) {
    SAETTA_REQUIRE(context_lens && new_lens && state.block_table && state.held && state.free_list && state.free_count && step.query_starts &&
                       step.kv_lens && step.slots && step.positions && step.unplaced,
                   SAETTA_E_NULL, "paged_tables: null buffer");
    for (const void *b : {static_cast<const void *>(context_lens), static_cast<const void *>(new_lens), static_cast<const void *>(state.block_table),
                          static_cast<const void *>(state.held), static_cast<const void *>(state.free_list), static_cast<const void *>(state.free_count),
                          static_cast<const void *>(step.query_starts), static_cast<const void *>(step.kv_lens), static_cast<const void *>(step.slots),
                          static_cast<const void *>(step.positions), static_cast<const void *>(step.unplaced)})
        SAETTA_REQUIRE(aligned(b, 4), SAETTA_E_ALIGN, "paged_tables: buffers must be 4-byte aligned");
    SAETTA_REQUIRE(block_tokens_ok(p.block_tokens), SAETTA_E_SHAPE, "paged_tables: blocks of %u tokens (16, 32, 64 or 128)", p.block_tokens);
    SAETTA_REQUIRE(p.blocks > 0 && uint64_t(p.blocks) * p.block_tokens < (1ull << 31), SAETTA_E_SHAPE,
                   "paged_tables: %u blocks of %u tokens (fewer than 2^31 tokens)", p.blocks, p.block_tokens);
    SAETTA_REQUIRE(p.max_blocks > 0 && uint64_t(p.max_blocks) * p.block_tokens < (1ull << 31), SAETTA_E_SHAPE, "paged_tables: rows of %u blocks", p.max_blocks);
    SAETTA_REQUIRE(p.requests < (1u << 24) && p.tokens < (1u << 31), SAETTA_E_SHAPE, "paged_tables: %u requests, room for %u tokens", p.requests, p.tokens);
    if (int rc = ensure_device()) return rc;
    const TablesArgs a = {context_lens, new_lens, state, step, p};
    // (one workgroup's slots: 1024 at a time)
    if (p.tokens <= 2 * TABLE_THREADS) {
        launch(paged_tables_kernel<true>, dim3(1), dim3(TABLE_THREADS), 0, as_stream(stream), a);
    } else {
        launch(paged_tables_kernel<false>, dim3(1), dim3(TABLE_THREADS), 0, as_stream(stream), a);
        launch(paged_slots_kernel, dim3((p.tokens + SLOT_TOKENS - 1) / SLOT_TOKENS), dim3(256), 0, as_stream(stream), a);
    }
    return launch_status("paged_tables");
}
