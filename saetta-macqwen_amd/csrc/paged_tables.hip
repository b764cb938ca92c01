// Block tables, slots and positions of a step, from the lengths of the requests.
//
// new'[r]: what of new[r] has room in the step, behind the requests before it.
// want[r] = min(ceil((context[r] + new'[r]) / block), max_blocks).  A request that holds fewer takes what is missing out of
// one segment at the end of the free list, request by request (an exclusive prefix sum of what they take); one that holds
// more gives the rest back behind what is left of the list, in the same order (another prefix sum).  So what a step takes
// and the next gives back whole leaves the list as it was.  The tokens' first rows are a third prefix sum.
//
// Bound by latency: a few bytes a request, two numbers a token.  The sums want every request, so one workgroup
// makes them, a request a thread, and moves the blocks' numbers, entry by entry over all its threads (a request is
// found by bisection in the prefix sums in LDS).  The tokens' slots are independent of each other: a second launch of as
// many workgroups as they fill, or, where few workgroups' worth of tokens come (a decode step), the first does them itself.
// Measured: 32 requests with a token and three drafts each 2.9 us; 512 requests of up to 1900 tokens admitted at once (8200 blocks, 126 thousand
// tokens) 8 us and 3 to 5 for the slots.
#include "common.hpp"
#include "lanes.hpp"
#include "paged_device.hpp"

namespace saetta {
namespace {

constexpr uint32_t SLOT_TOKENS = 256;  // of a workgroup of the second launch, one a thread
constexpr uint32_t AT_ONCE = 4;         // blocks' numbers that a thread has on their way (with 8 the same time)

struct TablesArgs {
    const uint32_t *context_lens, *new_lens;
    saetta_paged_state state;
    saetta_paged_step step;
    saetta_paged_tables_params p;
};

// Sums stop at the largest number there is (every order of adding gives the same).
__device__ __forceinline__ uint32_t add_up(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }

// Numbers summed over the threads before this one; `all`: over all of them.  (All threads; `waves` is free again on return.)
template <uint32_t TABLE_THREADS, int N>
__device__ __forceinline__ void sums_before(const uint32_t (&x)[N], uint32_t (*waves)[TABLE_THREADS / 64], uint32_t (&before)[N], uint32_t (&all)[N]) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t through[N];
#pragma unroll
    for (int i = 0; i < N; i++) through[i] = x[i];
#pragma unroll
    for (int d = 1; d < 64; d *= 2)
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t other = __shfl_up(through[i], d);
            if (lane >= uint32_t(d)) through[i] = add_up(through[i], other);
        }
#pragma unroll
    for (int i = 0; i < N; i++)
        if (lane == 63) waves[i][wave] = through[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        before[i] = all[i] = 0;
#pragma unroll
        for (uint32_t w = 0; w < TABLE_THREADS / 64; w++) {
            if (w == wave) before[i] = all[i];
            all[i] = add_up(all[i], waves[i][w]);
        }
        const uint32_t prior = __shfl_up(through[i], 1);
        before[i] = add_up(before[i], lane == 0 ? 0 : prior);
    }
    __syncthreads();
}

struct Lengths {
    uint32_t context, fresh, held, want;
};
__device__ __forceinline__ uint32_t blocks_of(const TablesArgs &a, uint32_t length) {
    const uint32_t bt = a.p.block_tokens;
    return min(length / bt + (length % bt != 0), a.p.max_blocks);
}
__device__ __forceinline__ Lengths lengths_of(const TablesArgs &a, uint32_t r) {
    Lengths l = {0, 0, 0, 0};
    if (r < a.p.requests) {
        l.context = a.context_lens[r], l.fresh = a.new_lens[r], l.held = min(a.state.held[r], a.p.max_blocks);
        // (of lengths that a step has left: tokens that it had no block for are counted in them and lie nowhere)
        if (a.context_lens == a.step.kv_lens) l.context = min(l.context, l.held * a.p.block_tokens);
        l.want = blocks_of(a, add_up(l.context, l.fresh));
    }
    return l;
}
// ... of a request whose first new token is token `token` of the step: those past the room are no part of it.
__device__ __forceinline__ void cut_to_room(const TablesArgs &a, uint32_t token, Lengths &l) {
    l.fresh = min(l.fresh, a.p.tokens - min(token, a.p.tokens));
    l.want = blocks_of(a, add_up(l.context, l.fresh));
}

// The same by a wave at once, 64 places a look, over memory.
__device__ __forceinline__ uint32_t wave_last_at_most(const uint32_t *starts, uint32_t n, uint32_t x) {
    uint32_t low = 0;
    const uint32_t lane = threadIdx.x & 63;
    while (n > 1) {
        const uint32_t each = (n + 63) / 64, at = lane * each;  // (lane 0's is one that is no more than x)
        const uint32_t found = 63 - uint32_t(__builtin_clzll(__ballot(at < n && (lane == 0 || starts[low + min(at, n - 1)] <= x)) | 1));
        low += found * each, n = min(each, n - found * each);
    }
    return low;
}

// Slot and position of token t of request r, `at` tokens behind the request's first, of a request that holds `held` blocks.
__device__ __forceinline__ void place_token(const TablesArgs &a, uint32_t t, uint32_t r, uint32_t at, uint32_t held) {
    const uint32_t bt = a.p.block_tokens, entry = at / bt;
    int32_t slot = -1;
    if (entry < held) {
        const uint32_t block = uint32_t(a.state.block_table[size_t(r) * a.p.max_blocks + entry]);
        if (block < a.p.blocks) slot = int32_t(block * bt + at % bt);
    }
    a.step.slots[t] = slot, a.step.positions[t] = int32_t(min(at, 0x7fffffffu));
}
__device__ __forceinline__ void place_nothing(const TablesArgs &a, uint32_t t) { a.step.slots[t] = a.step.positions[t] = -1; }

template <bool SLOTS, uint32_t TABLE_THREADS>
__global__ __launch_bounds__(TABLE_THREADS) void paged_tables_kernel(TablesArgs a) {
    __shared__ uint32_t waves[3][TABLE_THREADS / 64], starts[TABLE_THREADS], firsts[TABLE_THREADS], all_placed;
    // of a step of one round of requests: their first tokens, contexts and blocks, for the tokens' slots
    __shared__ uint32_t tokens_from[SLOTS ? TABLE_THREADS : 1], contexts[SLOTS ? TABLE_THREADS : 1], holds[SLOTS ? TABLE_THREADS : 1];
    const uint32_t tid = threadIdx.x, requests = a.p.requests, room = a.p.tokens;
    const uint32_t free_count = min(*a.state.free_count, a.p.blocks);

    if (tid == 0) all_placed = 0;
    auto take_of = [](const Lengths &l) { return l.want > l.held ? l.want - l.held : 0; };
    auto give_of = [](const Lengths &l) { return l.held > l.want ? l.held - l.want : 0; };

    // the step's tokens, and what is taken and given in all
    enum { TOKENS, TAKES, GIVES };
    uint32_t mine[3] = {0, 0, 0}, before[3], all[3];
    for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
        const Lengths l = lengths_of(a, r0 + tid);
        mine[TOKENS] = add_up(mine[TOKENS], l.fresh), mine[TAKES] = add_up(mine[TAKES], take_of(l)), mine[GIVES] = add_up(mine[GIVES], give_of(l));
    }
    sums_before<TABLE_THREADS>(mine, waves, before, all);
    const bool cut = all[TOKENS] > room, once = requests <= TABLE_THREADS && !cut;  // (once: the sums before a thread are those before its request)
    const uint32_t all_tokens = all[TOKENS], total = min(all_tokens, room);
    // Lengths of the request of this thread in a round, and the tokens before it: of a step past its room the sums of the tokens come first.
    auto lengths_in_room = [&](uint32_t r, uint32_t tokens_before) {
        Lengths l = lengths_of(a, r);
        if (cut) {
            const uint32_t fresh[1] = {l.fresh};
            uint32_t token[1], here[1];
            sums_before<TABLE_THREADS>(fresh, waves, token, here);
            if (r < requests) cut_to_room(a, add_up(tokens_before, token[0]), l);
        }
        return l;
    };
    if (cut) {
        mine[TAKES] = mine[GIVES] = 0;
        uint32_t tokens_before = 0;
        for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
            const Lengths l = lengths_in_room(r0 + tid, tokens_before);
            const uint32_t x[1] = {l.fresh};
            uint32_t none[1], here[1];
            sums_before<TABLE_THREADS>(x, waves, none, here);
            tokens_before = add_up(tokens_before, here[0]);
            mine[TAKES] = add_up(mine[TAKES], take_of(l)), mine[GIVES] = add_up(mine[GIVES], give_of(l));
        }
        sums_before<TABLE_THREADS>(mine, waves, before, all);
    }
    const uint32_t taken = min(all[TAKES], free_count), left = free_count - taken, all_gives = all[GIVES];

    // blocks that are taken; the requests' first tokens and lengths
    uint32_t takes_before = 0, tokens_before = 0, placed = 0;
    for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
        const uint32_t r = r0 + tid;
        const Lengths l = lengths_in_room(r, tokens_before);
        const uint32_t take = take_of(l), x[2] = {l.fresh, take};
        uint32_t first_of[2] = {before[TOKENS], before[TAKES]}, of_all[2] = {all[TOKENS], all[TAKES]};
        if (!once) sums_before<TABLE_THREADS>(x, waves, first_of, of_all);
        const uint32_t token = add_up(tokens_before, first_of[TOKENS]), here = of_all[TAKES], before_it = add_up(takes_before, first_of[TAKES]);
        tokens_before = add_up(tokens_before, of_all[TOKENS]), takes_before = add_up(takes_before, here);
        if (r < requests) {
            a.step.query_starts[r] = min(token, room);
            a.step.kv_lens[r] = add_up(l.context, l.fresh);
            const uint32_t held = l.held + min(take, taken - min(before_it, taken));
            if (take > 0) a.state.held[r] = held;
            // tokens that its blocks have places for
            const uint32_t places = min(held, l.want) * a.p.block_tokens;
            if (l.context < places) placed += min(l.fresh, places - l.context);
            if constexpr (SLOTS) tokens_from[tid] = min(token, room), contexts[tid] = l.context, holds[tid] = min(held, l.want);
        }
        if (here == 0) continue;  // (for all threads alike)
        starts[tid] = before_it, firsts[tid] = l.held;
        __syncthreads();
        const uint32_t first = starts[0], end = min(takes_before, taken), n = min(TABLE_THREADS, requests - r0);
        for (uint32_t k0 = first + tid; k0 < end; k0 += AT_ONCE * TABLE_THREADS) {
            uint32_t k[AT_ONCE], of[AT_ONCE];
            int32_t block[AT_ONCE];
#pragma unroll
            for (uint32_t j = 0; j < AT_ONCE; j++) k[j] = min(k0 + j * TABLE_THREADS, end - 1), block[j] = a.state.free_list[left + k[j]];
            last_at_most(starts, n, k, of);
#pragma unroll
            for (uint32_t j = 0; j < AT_ONCE; j++)
                if (k0 + j * TABLE_THREADS < end) a.state.block_table[size_t(r0 + of[j]) * a.p.max_blocks + firsts[of[j]] + (k[j] - starts[of[j]])] = block[j];
        }
        __syncthreads();
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) placed += __shfl_xor(placed, d);
    if ((tid & 63) == 0 && placed) atomicAdd(&all_placed, placed);
    __syncthreads();  // (and what is taken has been read: what is given may land there)
    if (tid == 0) {
        *a.step.unplaced = all_tokens - all_placed;
        a.step.query_starts[requests] = total;
        *a.state.free_count = min(add_up(left, all_gives), a.p.blocks);
    }

    if (all_gives > 0) {
        uint32_t gives_before = 0;
        for (uint32_t r0 = 0; r0 < requests; r0 += TABLE_THREADS) {
            const uint32_t r = r0 + tid;
            // (lengths from kv_lens: context_lens may be the same array)
            Lengths l = {0, 0, 0, 0};
            if (r < requests) {
                l.held = min(a.state.held[r], a.p.max_blocks);
                l.want = blocks_of(a, a.step.kv_lens[r]);
            }
            const uint32_t give = l.held > l.want ? l.held - l.want : 0;
            const uint32_t x[1] = {give};
            uint32_t first_of[1], here[1];
            sums_before<TABLE_THREADS>(x, waves, first_of, here);
            starts[tid] = add_up(gives_before, first_of[0]), firsts[tid] = l.want;
            gives_before = add_up(gives_before, here[0]);
            if (here[0] == 0) continue;
            __syncthreads();
            const uint32_t first = starts[0], n = min(TABLE_THREADS, requests - r0);
            for (uint32_t k0 = first + tid; k0 < gives_before; k0 += AT_ONCE * TABLE_THREADS) {
                uint32_t k[AT_ONCE], of[AT_ONCE];
                int32_t *entry[AT_ONCE], block[AT_ONCE];
#pragma unroll
                for (uint32_t j = 0; j < AT_ONCE; j++) k[j] = min(k0 + j * TABLE_THREADS, gives_before - 1);
                last_at_most(starts, n, k, of);
#pragma unroll
                for (uint32_t j = 0; j < AT_ONCE; j++) {
                    entry[j] = a.state.block_table + size_t(r0 + of[j]) * a.p.max_blocks + firsts[of[j]] + (k[j] - starts[of[j]]);
                    block[j] = *entry[j];
                }
#pragma unroll
                for (uint32_t j = 0; j < AT_ONCE; j++) {
                    if (k0 + j * TABLE_THREADS >= gives_before) break;
                    // (more than the list has room for: a table that names blocks twice; they are lost, not written past its end)
                    if (left + k[j] < a.p.blocks) a.state.free_list[left + k[j]] = block[j];
                    *entry[j] = -1;
                }
            }
            __syncthreads();
            if (give > 0) a.state.held[r] = l.want;
        }
    }

    if constexpr (SLOTS) {
        __syncthreads();
        for (uint32_t t = tid; t < room; t += TABLE_THREADS) {
            if (t < total) {
                // (requests without new tokens share their start with the next: the last of them is the token's)
                const uint32_t r = last_at_most(tokens_from, requests, t);
                place_token(a, t, r, add_up(contexts[r], t - tokens_from[r]), holds[r]);
            } else {
                place_nothing(a, t);
            }
        }
    }
}

// The second launch: SLOT_TOKENS tokens a workgroup.  The requests that they belong to are those between the first token's and the last's.
__global__ __launch_bounds__(SLOT_TOKENS) void paged_slots_kernel(TablesArgs a) {
    constexpr uint32_t HELD = 1024;
    __shared__ uint32_t starts[HELD];
    const uint32_t *query_starts = a.step.query_starts, total = query_starts[a.p.requests], t0 = blockIdx.x * SLOT_TOKENS;
    uint32_t first = 0, n = 1;
    if (t0 < total) {
        first = wave_last_at_most(query_starts, a.p.requests, t0);
        n = first + wave_last_at_most(query_starts + first, a.p.requests - first, min(t0 + SLOT_TOKENS, total) - 1) + 1 - first;
        for (uint32_t i = threadIdx.x; i < min(n, HELD); i += SLOT_TOKENS) starts[i] = query_starts[first + i];
    }
    __syncthreads();
    const uint32_t t = t0 + threadIdx.x;
    if (t < total) {
        const uint32_t r = first + (n <= HELD ? last_at_most(starts, n, t) : last_at_most(query_starts + first, n, t));
        // (the context from the sum and not from context_lens, which kv_lens may be: those have grown by now)
        const uint32_t context = a.step.kv_lens[r] - (query_starts[r + 1] - query_starts[r]);
        place_token(a, t, r, add_up(context, t - query_starts[r]), min(a.state.held[r], a.p.max_blocks));
    } else if (t < a.p.tokens) {
        place_nothing(a, t);
    }
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
    SAETTA_REQUIRE(uint64_t(p.requests) * p.max_blocks < (1ull << 31), SAETTA_E_SHAPE, "paged_tables: a table of %u rows of %u blocks (fewer than 2^31 entries)", p.requests, p.max_blocks);
    SAETTA_REQUIRE(p.requests < (1u << 24) && p.tokens < (1u << 31), SAETTA_E_SHAPE, "paged_tables: %u requests, room for %u tokens", p.requests, p.tokens);
    if (int rc = ensure_device()) return rc;
    const TablesArgs a = {context_lens, new_lens, state, step, p};
    // One workgroup's slots, of requests that it has in LDS, or two launches.  A small step's workgroup is four waves, whose barriers are cheaper.
    if (p.tokens <= 512 && p.requests <= 256) {
        launch(paged_tables_kernel<true, 256>, dim3(1), dim3(256), 0, as_stream(stream), a);
    } else if (p.tokens <= 2048 && p.requests <= 1024) {
        launch(paged_tables_kernel<true, 1024>, dim3(1), dim3(1024), 0, as_stream(stream), a);
    } else {
        launch(paged_tables_kernel<false, 1024>, dim3(1), dim3(1024), 0, as_stream(stream), a);
        if (p.tokens > 0) launch(paged_slots_kernel, dim3((p.tokens + SLOT_TOKENS - 1) / SLOT_TOKENS), dim3(SLOT_TOKENS), 0, as_stream(stream), a);
    }
    return launch_status("paged_tables");
}
