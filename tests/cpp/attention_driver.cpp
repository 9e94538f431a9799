// Writes keys and values into a cache, reads them back and attends to them through the C++20 host side.
//   attention_driver case.bin result.bin
// case.bin: uint64 {prompts, images, keys, tokens, heads, head_dim, dtype}, then FP16 keys and values
// [prompts, keys, heads, head_dim] and queries [images, tokens, heads, head_dim]. result.bin: keys and values as read back, then
// the output, all FP16.
#include "sdxlq_ops.hpp"

#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <stdexcept>
#include <vector>

namespace {

void check(cudaError_t error) {
    if (error != cudaSuccess) throw std::runtime_error(cudaGetErrorString(error));
}

struct Buffer {
    void* data = nullptr;
    explicit Buffer(std::size_t bytes) { check(cudaMalloc(&data, bytes)); }
    ~Buffer() { cudaFree(data); }
    Buffer(const Buffer&) = delete;
    Buffer& operator=(const Buffer&) = delete;
};

void load(std::FILE* file, void* device, std::size_t bytes) {
    std::vector<char> host(bytes);
    if (std::fread(host.data(), 1, bytes, file) != bytes) throw std::runtime_error("short case file");
    check(cudaMemcpy(device, host.data(), bytes, cudaMemcpyHostToDevice));
}

void store(std::FILE* file, const void* device, std::size_t bytes) {
    std::vector<char> host(bytes);
    check(cudaMemcpy(host.data(), device, bytes, cudaMemcpyDeviceToHost));
    if (std::fwrite(host.data(), 1, bytes, file) != bytes) throw std::runtime_error("short result file");
}

}  // namespace

int main(int argc, char** argv) try {
    if (argc != 3) return 2;
    std::FILE* const in = std::fopen(argv[1], "rb");
    std::FILE* const out = std::fopen(argv[2], "wb");
    if (in == nullptr || out == nullptr) return 2;
    uint64_t n[7];
    if (std::fread(n, sizeof(n), 1, in) != 1) return 2;
    const uint64_t prompts = n[0], images = n[1], keys = n[2], tokens = n[3], heads = n[4], dim = n[5];
    const std::size_t kv = prompts * keys * heads * dim, q = images * tokens * heads * dim;
    Buffer k(kv * 2), v(kv * 2), query(q * 2), y(q * 2), held_k(kv * 2), held_v(kv * 2), k_scales(prompts * heads * keys * 4),
        v_scales(prompts * heads * keys * 4);
    load(in, k.data, kv * 2);
    load(in, v.data, kv * 2);
    load(in, query.data, q * 2);

    sdxlq::Runtime runtime(0, nullptr, 64u << 20);
    const sdxlq::Ops ops(runtime, nullptr);
    sdxlq_kv_cache cache{};
    cache.k = held_k.data;
    cache.v = held_v.data;
    cache.dtype = static_cast<int32_t>(n[6]);
    if (cache.dtype != SDXLQ_FP16) {
        cache.k_scales = static_cast<float*>(k_scales.data);
        cache.v_scales = static_cast<float*>(v_scales.data);
    }
    cache.slots = prompts;
    cache.capacity = keys;
    cache.heads = heads;
    cache.head_dim = dim;
    cache.slot_stride = heads * keys * dim;
    cache.token_stride = dim;
    cache.head_stride = keys * dim;
    sdxlq_kv_tokens rows{};
    rows.k = k.data;
    rows.v = v.data;
    rows.rows = prompts;
    rows.tokens = keys;
    rows.row_stride = keys * heads * dim;
    rows.token_stride = heads * dim;
    rows.head_stride = dim;
    ops.kv_cache_write(cache, rows);
    ops.kv_cache_read(cache, rows);          // in the place of what was written

    sdxlq_attention_desc desc{};
    desc.q = query.data;
    desc.y = y.data;
    desc.batch = images;
    desc.q_tokens = tokens;
    desc.q_heads = heads;
    desc.head_dim = dim;
    desc.q_batch_stride = desc.y_batch_stride = tokens * heads * dim;
    desc.q_token_stride = desc.y_token_stride = heads * dim;
    desc.q_head_stride = desc.y_head_stride = dim;
    desc.prefix = cache;
    desc.scale = 1.0f / std::sqrt(static_cast<float>(dim));
    ops.shared_prefix_attention(desc);
    desc.prefix.slots = images + 1;
    bool refused = false;
    try {
        ops.shared_prefix_attention(desc);
    } catch (const sdxlq::CudaError&) {
        refused = true;
    }
    if (!refused) throw std::runtime_error("a batch that is no multiple of its prefixes was not refused");
    check(cudaDeviceSynchronize());
    store(out, k.data, kv * 2);
    store(out, v.data, kv * 2);
    store(out, y.data, q * 2);
    std::fclose(in);
    std::fclose(out);
    return 0;
} catch (const std::exception& error) {
    std::fprintf(stderr, "%s\n", error.what());
    return 1;
}
