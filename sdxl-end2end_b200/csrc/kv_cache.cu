// Writing FP16 keys and values into a cache of INT8, FP8 or FP16 elements, and reading them back.
//
// The vector of one token and one head, x[D], is quantised by itself, with a = max |x_d| over finite values:
//   INT8  s = fp32(a / 127), q = clamp(rne(x / s), -127, 127), NaN -> 0
//   FP8   s = 2^e, the smallest with a / s at most the format's largest value; q = rne(x / s), saturating
//   a = 0 gives s = 1 in both.
// and read back as fp16(q s). The FP8 scale is a power of two, so that x / s and q s are exact and the only rounding
// is the format's own; in a floating-point format it costs no precision, only a share of an octave of range. rne(x / s) for
// INT8 is that of the exact quotient: r = rne(x * (1 / s)) is at most one off, and the remainder x - r s, exact in
// one fused multiply-add (r s and x are multiples of units that keep it within 24 bits), says to which side.
//
// What bounds it: memory for large copies, latency for small ones. A lane takes 16 bytes of K and of V of one vector, D / 8
// lanes share a vector's maximum by shuffles. The block's vectors run over tokens first: the FP16 side is then read in
// whole 128-byte lines and the cache, whose tokens of one head lie behind one another, is written in runs.

#include "attention.cuh"

namespace sdxlq {

namespace {

constexpr uint32_t kThreads = 256;

// Largest finite magnitude of eight halves.
__device__ __forceinline__ float largest_finite(const uint4 raw) { return finite_max(raw, 0.0f); }

// Scale of a vector and the factor that divides by it: exact for FP8, for INT8 the rounded reciprocal.
template <int kFormat>
__device__ __forceinline__ float2 scale_of(float maximum) {
    if (maximum == 0.0f) return make_float2(1.0f, 1.0f);
    if constexpr (kFormat == KV_INT8) {
        const float scale = __fdiv_rn(maximum, 127.0f);
        return make_float2(scale, __fdiv_rn(1.0f, scale));
    } else {
        // the format's largest value is 1.75 * 2^8 or 1.75 * 2^15; an FP16 maximum is a normal FP32 number
        const uint32_t bits = __float_as_uint(maximum);
        const int top = kFormat == KV_E4M3 ? 8 : 15;
        const int exponent = static_cast<int>(bits >> 23) - 127 - top + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
        return make_float2(__uint_as_float(static_cast<uint32_t>(127 + exponent) << 23),
                           __uint_as_float(static_cast<uint32_t>(127 - exponent) << 23));
    }
}

// clamp(rne(x / scale), -127, 127) of the exact quotient; NaN -> 0.
__device__ __forceinline__ uint32_t quantise_exact(float x, float2 scale) {
    float r = rintf(x * scale.y);
    const float rest = fmaf(-r, scale.x, x), half_step = 0.5f * scale.x;
    const bool odd = (static_cast<int>(r) & 1) != 0;
    if (rest > half_step || (rest == half_step && odd)) r += 1.0f;
    if (rest < -half_step || (rest == -half_step && odd)) r -= 1.0f;
    return quantize_s8(r < -127.0f ? -127.0f : r);
}

template <int kFormat>
__device__ __forceinline__ uint2 encode_vector(const uint4 raw, float2 scale) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t out[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (kFormat == KV_INT8) {
            out[i] = pack_bytes(quantise_exact(half_lo(words[2 * i]), scale), quantise_exact(half_hi(words[2 * i]), scale),
                                quantise_exact(half_lo(words[2 * i + 1]), scale), quantise_exact(half_hi(words[2 * i + 1]), scale));
        } else {
            const uint32_t fmt = kFormat == KV_E4M3 ? 0u : 1u;
            out[i] = encode_fp8x2(half_lo(words[2 * i]) * scale.y, half_hi(words[2 * i]) * scale.y, fmt) |
                     (encode_fp8x2(half_lo(words[2 * i + 1]) * scale.y, half_hi(words[2 * i + 1]) * scale.y, fmt) << 16);
        }
    }
    return make_uint2(out[0], out[1]);
}

// fp16(q scale), saturating: rounding up to the format's grid can pass the largest half.
__device__ __forceinline__ uint32_t scaled_pair(uint32_t pair, float scale) {
    const __half2 h = as_half2(pair);
    const float lo = __low2float(h) * scale, hi = __high2float(h) * scale;
    const auto within = [](float x) { return x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x; };
    return pack_half2(within(lo), within(hi));
}

template <int kFormat>
__device__ __forceinline__ uint4 decode_vector(const uint2 bytes, float scale) {
    const uint2 a = widen4<kFormat>(bytes.x), b = widen4<kFormat>(bytes.y);
    return make_uint4(scaled_pair(a.x, scale), scaled_pair(a.y, scale), scaled_pair(b.x, scale), scaled_pair(b.y, scale));
}

struct Geometry {
    uint32_t lanes_log2;         // lanes of a vector: the power of two at or above dim / 8
    uint32_t tokens_log2;        // tokens of a block; its other vectors are heads
    uint32_t token_tiles, head_tiles;
};

template <int kFormat, bool kWrite>
__global__ void __launch_bounds__(kThreads) kv_copy_kernel(const __grid_constant__ KvCopyLaunch p, const Geometry geometry) {
    wait_for_prior_kernels_then_release_next();
    const uint32_t lane = threadIdx.x & ((1u << geometry.lanes_log2) - 1u), vector = threadIdx.x >> geometry.lanes_log2;
    const uint32_t token_tile = blockIdx.x % geometry.token_tiles, rest = blockIdx.x / geometry.token_tiles;
    const uint32_t head_tile = rest % geometry.head_tiles, row = rest / geometry.head_tiles;
    const uint32_t block_heads = (kThreads >> geometry.lanes_log2) >> geometry.tokens_log2;
    const uint32_t token = (token_tile << geometry.tokens_log2) + (vector & ((1u << geometry.tokens_log2) - 1u));
    const uint32_t head = head_tile * block_heads + (vector >> geometry.tokens_log2);
    const bool live = lane * 8u < p.dim && token < p.tokens && head < p.heads;

    const int64_t first = p.positions != nullptr ? __ldg(p.positions + row) : static_cast<int64_t>(p.start);
    const int64_t at = first + token;
    const int64_t count = p.counts != nullptr ? __ldg(p.counts + row) : static_cast<int64_t>(p.tokens);
    const bool present = live && token < count && at >= 0 && at < p.cache.capacity;

    const int64_t outside = row * p.row_stride + token * p.token_stride + head * p.head_stride + lane * 8u;
    const uint32_t slot = p.first_slot + row;
    const int64_t width = kFormat == KV_F16 ? 2 : 1;
    const int64_t inside = slot * p.cache.slot_stride + at * p.cache.token_stride + head * p.cache.head_stride + lane * 8u * width;
    const int64_t scale_at = (static_cast<int64_t>(slot) * p.heads + head) * p.cache.capacity + at;

    if constexpr (kWrite) {
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        if (present) {
            k = __ldg(reinterpret_cast<const uint4*>(p.k + outside));
            v = __ldg(reinterpret_cast<const uint4*>(p.v + outside));
        }
        if constexpr (kFormat == KV_F16) {
            if (present) {
                *reinterpret_cast<uint4*>(p.cache.k + inside) = k;
                *reinterpret_cast<uint4*>(p.cache.v + inside) = v;
            }
        } else {
            float k_max = largest_finite(k), v_max = largest_finite(v);
            for (uint32_t offset = 1; offset < (1u << geometry.lanes_log2); offset <<= 1) {
                k_max = fmaxf(k_max, __shfl_xor_sync(0xffffffffu, k_max, offset));
                v_max = fmaxf(v_max, __shfl_xor_sync(0xffffffffu, v_max, offset));
            }
            const float2 k_scale = scale_of<kFormat>(k_max), v_scale = scale_of<kFormat>(v_max);
            if (present) {
                *reinterpret_cast<uint2*>(p.cache.k + inside) = encode_vector<kFormat>(k, k_scale);
                *reinterpret_cast<uint2*>(p.cache.v + inside) = encode_vector<kFormat>(v, v_scale);
                if (lane == 0) {
                    p.cache.k_scales[scale_at] = k_scale.x;
                    p.cache.v_scales[scale_at] = v_scale.x;
                }
            }
        }
    } else {
        uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
        if (present) {
            if constexpr (kFormat == KV_F16) {
                k = __ldg(reinterpret_cast<const uint4*>(p.cache.k + inside));
                v = __ldg(reinterpret_cast<const uint4*>(p.cache.v + inside));
            } else {
                const uint2 k_bytes = __ldg(reinterpret_cast<const uint2*>(p.cache.k + inside));
                const uint2 v_bytes = __ldg(reinterpret_cast<const uint2*>(p.cache.v + inside));
                k = decode_vector<kFormat>(k_bytes, __ldg(p.cache.k_scales + scale_at));
                v = decode_vector<kFormat>(v_bytes, __ldg(p.cache.v_scales + scale_at));
            }
        }
        if (live) {
            *reinterpret_cast<uint4*>(p.k + outside) = k;
            *reinterpret_cast<uint4*>(p.v + outside) = v;
        }
    }
}

uint32_t log2_at_least(uint32_t value) {
    uint32_t log2 = 0;
    while ((1u << log2) < value) ++log2;
    return log2;
}

template <bool kWrite>
cudaError_t launch_copy(const KvCopyLaunch& launch, cudaStream_t stream, bool early_launch) {
    Geometry geometry{};
    geometry.lanes_log2 = log2_at_least(launch.dim / 8);
    const uint32_t vectors_log2 = 8 - geometry.lanes_log2;
    geometry.tokens_log2 = log2_at_least(launch.tokens);
    if (geometry.tokens_log2 > vectors_log2) geometry.tokens_log2 = vectors_log2;
    const uint32_t tokens = 1u << geometry.tokens_log2, heads = 1u << (vectors_log2 - geometry.tokens_log2);
    geometry.token_tiles = (launch.tokens + tokens - 1) / tokens;
    geometry.head_tiles = (launch.heads + heads - 1) / heads;
    const uint64_t blocks = static_cast<uint64_t>(geometry.token_tiles) * geometry.head_tiles * launch.rows;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    const auto run = [&](auto kernel) { return launch_behind(kernel, static_cast<uint32_t>(blocks), kThreads, 0, stream, early_launch, launch, geometry); };
    switch (launch.format) {
    case KV_E4M3: return run(kv_copy_kernel<KV_E4M3, kWrite>);
    case KV_E5M2: return run(kv_copy_kernel<KV_E5M2, kWrite>);
    case KV_INT8: return run(kv_copy_kernel<KV_INT8, kWrite>);
    default: return run(kv_copy_kernel<KV_F16, kWrite>);
    }
}

}  // namespace

cudaError_t launch_kv_write(const KvCopyLaunch& launch, cudaStream_t stream, bool early_launch) {
    return launch_copy<true>(launch, stream, early_launch);
}

cudaError_t launch_kv_read(const KvCopyLaunch& launch, cudaStream_t stream, bool early_launch) {
    return launch_copy<false>(launch, stream, early_launch);
}

}  // namespace sdxlq
