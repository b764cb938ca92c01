// The paged cache of the C++ host mirror (saetta-macqwen_amd/host/saetta.hpp, namespace paged) as a program uses it: tables, store
// and attention recorded as a plan and replayed from a graph, against the formula in 64 bits over what the cache gives back.
// Exit code 0 = all passed.  Run by tests/test_gpu_paged_host_cpp.py on a GPU box.
#include <cstdio>

#include "../../saetta-macqwen_amd/host/saetta.hpp"

using namespace saetta;

static int failures = 0;
#define EXPECT(cond, ...)                      \
    do {                                       \
        if (!(cond)) {                         \
            failures++;                        \
            std::printf("FAIL: " __VA_ARGS__); \
            std::printf("\n");                 \
        }                                      \
    } while (0)

constexpr size_t HEADS = 16, KV = 2, DIM = 256, REQUESTS = 3, ROOM = 24, BLOCK = 16, BLOCKS = 30;

static std::vector<_Float16> noise(size_t n, uint32_t seed) {
    std::vector<_Float16> x(n);
    uint32_t s = seed * 2654435761u + 1;
    for (auto &v : x) {
        float sum = 0.0f;
        for (int i = 0; i < 4; i++) s = s * 1664525u + 1013904223u, sum += float(s >> 8) / float(1 << 24) - 0.5f;
        v = _Float16(sum * 1.7f);
    }
    return x;
}
template <class T>
static void upload(const gpu::Buffer &b, const std::vector<T> &x) {
    hip_check(hipMemcpy(b.get(), x.data(), x.size() * sizeof(T), hipMemcpyHostToDevice), "hipMemcpy");
}

int main() {
    gpu::Gpu gpu;
    const paged::PagedCache cache(gpu, KV, DIM, BLOCKS, BLOCK);
    const paged::PagedTables tables(gpu, REQUESTS, ROOM, 12, BLOCKS, BLOCK);
    const paged::PagedAttention attention(gpu, HEADS, KV, DIM, tables, 17);
    const gpu::Buffer context = gpu.buffer(REQUESTS * 4), fresh = gpu.buffer(REQUESTS * 4);
    const size_t ROW = HEADS + 2 * KV;  // q, k and v of a projection side by side
    const gpu::Buffer qkv = gpu.buffer(ROOM * ROW * DIM * 2), out = gpu.buffer(ROOM * HEADS * DIM * 2);
    const paged::Rows q(View(qkv), ROW * DIM, DIM), k(View(qkv, HEADS * DIM * 2), ROW * DIM, DIM), v(View(qkv, (HEADS + KV) * DIM * 2), ROW * DIM, DIM);
    plan::Plan plan(gpu);
    tables.record(plan, View(context), View(fresh));
    cache.record(plan, paged::Type::F16, k, v, View(tables.slots), ROOM);
    attention.record_split(plan);
    attention.record(plan, paged::Type::F16, q, cache, paged::Rows(View(out), HEADS));
    const plan::Built built = plan.build(true);

    std::vector<uint32_t> lengths(REQUESTS, 0);
    const uint32_t steps[4][REQUESTS] = {{17, 0, 5}, {1, 4, 1}, {2, 2, 0}, {1, 17, 1}};
    for (int step = 0; step < 4; step++) {
        const std::vector<uint32_t> now(steps[step], steps[step] + REQUESTS);
        upload(context, lengths), upload(fresh, now);
        const auto x = noise(ROOM * ROW * DIM, step + 1);
        upload(qkv, x);
        built.run(gpu);
        gpu.sync();
        const auto table = gpu::contents<int32_t>(tables.block_table, REQUESTS * 12);
        const auto got = gpu::contents<_Float16>(out, ROOM * HEADS * DIM);
        double worst = 0.0;
        size_t row = 0;
        for (size_t r = 0; r < REQUESTS; r++) {
            const size_t n = lengths[r] + now[r];
            if (now[r] == 0) continue;
            // what the request's slots hold
            std::vector<int32_t> slots(n);
            for (size_t t = 0; t < n; t++) slots[t] = table[r * 12 + t / BLOCK] * int32_t(BLOCK) + int32_t(t % BLOCK);
            const gpu::Buffer s = gpu.buffer_from(slots), kb = gpu.buffer(n * KV * DIM * 4), vb = gpu.buffer(n * KV * DIM * 4);
            cache.encode_dequantize(gpu, paged::Type::F32, View(s), View(kb), View(vb), n);
            gpu.sync();
            const auto keys = gpu::contents<float>(kb, n * KV * DIM), values = gpu::contents<float>(vb, n * KV * DIM);
            for (size_t i = 0; i < now[r]; i++, row++) {
                // the newest key is the one that was given, to half a step of e4m3 (2^-4) of it or of the block's smallest step
                for (size_t d = 0; d < KV * DIM; d++) {
                    const float want = float(x[(row * ROW + HEADS) * DIM + d]), is = keys[(lengths[r] + i) * KV * DIM + d];
                    EXPECT(std::fabs(is - want) <= std::fabs(want) / 16 + 1e-4f, "step %d request %zu token %zu: key %g, stored %g", step, r, i, want, is);
                }
                for (size_t h = 0; h < HEADS; h++) {
                    const size_t seen = lengths[r] + i + 1, kv = h / (HEADS / KV);
                    std::vector<double> p(seen);
                    double top = -1e300, sum = 0.0;
                    for (size_t t = 0; t < seen; t++) {
                        double dot = 0.0;
                        for (size_t d = 0; d < DIM; d++) dot += double(x[(row * ROW + h) * DIM + d]) * keys[(t * KV + kv) * DIM + d];
                        p[t] = dot / 16.0, top = std::max(top, p[t]);
                    }
                    for (auto &w : p) w = std::exp(w - top), sum += w;
                    for (size_t d = 0; d < DIM; d++) {
                        double o = 0.0, size = 0.0;
                        for (size_t t = 0; t < seen; t++) o += p[t] / sum * values[(t * KV + kv) * DIM + d], size += p[t] / sum * std::fabs(values[(t * KV + kv) * DIM + d]);
                        // weights in f16 (2^-11 of what they weigh), sums in f32, the output in f16 (2^-11 of it)
                        const double off = std::fabs(double(got[(row * HEADS + h) * DIM + d]) - o);
                        worst = std::max(worst, off / (size * 0x1p-11 * 1.1 + std::fabs(o) * 0x1p-11 + 0x1p-24));
                    }
                }
            }
        }
        std::printf("step %d: %zu rows, at most %.2f of the bound\n", step, row, worst);
        EXPECT(worst <= 1.0, "step %d: %.2f of the bound", step, worst);
        for (size_t r = 0; r < REQUESTS; r++) lengths[r] += now[r];
        if (step == 2) lengths[0] -= 1, lengths[2] = 0;  // a rejected token; a finished request
    }
    for (int bad = 0; bad < 3; bad++) {
        bool threw = false;
        try {
            if (bad == 0) paged::PagedCache(gpu, KV, 128, BLOCKS, BLOCK);
            if (bad == 1) paged::PagedCache(gpu, KV, DIM, BLOCKS, 24);
            if (bad == 2) paged::PagedAttention(gpu, 24, KV, DIM, tables, 1);
        } catch (const std::runtime_error &) {
            threw = true;
        }
        EXPECT(threw, "refusal %d", bad);
    }
    std::printf(failures ? "%d FAILURES\n" : "all paged host tests passed\n", failures);
    return failures ? 1 : 0;
}
