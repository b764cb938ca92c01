// What the paged objects of the C++ host mirror refuse of sizes that 32 bits do not hold: cut to them they would be another call's.
// Exit code 0 = all passed.  Run by tests/test_gpu_paged_host_cpp_sizes.py on a GPU.
#include <cstdio>

#include "../../saetta-macqwen_amd/host/saetta.hpp"

using namespace saetta;

template <class F>
static int refused(const char *what, F f) {
    try {
        f();
    } catch (const std::runtime_error &e) {
        if (std::string(e.what()).find("2^32") != std::string::npos) return 0;
        std::printf("FAIL: %s: %s\n", what, e.what());
        return 1;
    }
    std::printf("FAIL: %s was taken\n", what);
    return 1;
}

int main() {
    gpu::Gpu gpu;
    const size_t MUCH = (size_t(1) << 32) + 1;
    const paged::PagedTables tables(gpu, 2, 4, 3, 6, 16);
    const paged::PagedCache cache(gpu, 2, 256, 6, 16);
    const gpu::Buffer rows = gpu.buffer(2 * 256 * 4), slots = gpu.buffer(4);
    const paged::Rows k(View(rows), 2);
    int failures = 0;
    failures += refused("rows", [&] { paged::PagedAttention(gpu, 16, 2, 256, tables, MUCH); });
    failures += refused("heads", [&] { paged::PagedAttention(gpu, MUCH + 15, MUCH + 1, 256, tables, 1); });
    failures += refused("requests", [&] { paged::PagedTables(gpu, MUCH, 4, 3, 6, 16); });
    failures += refused("tokens", [&] { paged::PagedTables(gpu, 2, MUCH, 3, 6, 16); });
    failures += refused("kv heads", [&] { paged::PagedCache(gpu, MUCH, 256, 6, 16); });
    failures += refused("a store's tokens", [&] { cache.encode(gpu, paged::Type::F32, k, k, View(slots), MUCH); });
    failures += refused("a gather's tokens", [&] { cache.encode_dequantize(gpu, paged::Type::F32, View(slots), View(rows), View(rows), MUCH); });
    std::printf(failures ? "%d FAILURES\n" : "all sizes refused\n", failures);
    return failures ? 1 : 0;
}
