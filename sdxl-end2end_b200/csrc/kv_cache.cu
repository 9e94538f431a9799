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
// What bounds it: memory for large copies (16 x 4096 tokens of 10 heads of 64 into INT8 and back: 106 us, 4.8 TB/s), latency for
// small ones (2 x 77 tokens: 4 us a launch). A lane takes 16 bytes of K and of V of one vector, D / 8
// lanes share a vector's maximum by shuffles. The block's vectors run over tokens first: the FP16 side is then read in
// whole 128-byte lines and the cache, whose tokens of one head lie behind one another, is written in runs.

#include "attention.cuh"

#include <type_traits>

namespace sdxlq {

namespace {

constexpr uint32_t kThreads = 256;

// Largest finite magnitude of eight halves.
__device__ __forceinline__ float largest_finite(const uint4 raw) {
    const __half2 a = __hmax2(__habs2(as_half2(raw.x)), __habs2(as_half2(raw.y))), b = __hmax2(__habs2(as_half2(raw.z)), __habs2(as_half2(raw.w)));
    const __half2 c = __hmax2(a, b);
    const float largest = fmaxf(__low2float(c), __high2float(c));        // NaN never wins
    return largest <= 65504.0f ? largest : finite_max(raw, 0.0f);
}

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

__device__ __forceinline__ float max3_nan(float a, float b, float c) {
    float y;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

// Eight values at once. Adding 1.5 * 2^23 rounds x * (1 / s) and leaves the integer in the sum's low byte; where a remainder is
// half a step or more (or a value is not finite), the vector is taken one value at a time.
__device__ __forceinline__ uint2 encode_int8(const uint4 raw, float2 scale) {
    const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
    const float2 inverse = make_float2(scale.y, scale.y), step = make_float2(-scale.x, -scale.x), magic = make_float2(12582912.0f, 12582912.0f);
    uint32_t bytes[8];
    float largest = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(as_half2(words[i]));
        const float2 sum = __fadd2_rn(__fmul2_rn(x, inverse), magic);
        const float2 rest = __ffma2_rn(__fadd2_rn(sum, make_float2(-12582912.0f, -12582912.0f)), step, x);
        largest = max3_nan(largest, fabsf(rest.x), fabsf(rest.y));
        bytes[2 * i] = __float_as_uint(sum.x);
        bytes[2 * i + 1] = __float_as_uint(sum.y);
    }
    if (!(largest < 0.5f * scale.x)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bytes[2 * i] = quantise_exact(half_lo(words[i]), scale);
            bytes[2 * i + 1] = quantise_exact(half_hi(words[i]), scale);
        }
    }
    return make_uint2(pack_bytes(bytes[0], bytes[1], bytes[2], bytes[3]), pack_bytes(bytes[4], bytes[5], bytes[6], bytes[7]));
}

template <int kFormat>
__device__ __forceinline__ uint2 encode_vector(const uint4 raw, float2 scale) {
    if constexpr (kFormat == KV_INT8) {
        return encode_int8(raw, scale);
    } else {
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
        const uint32_t fmt = kFormat == KV_E4M3 ? 0u : 1u;
        uint32_t out[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 x = __fmul2_rn(__half22float2(as_half2(words[i])), make_float2(scale.y, scale.y));
            out[i] = encode_fp8x2(x.x, x.y, fmt);
        }
        return make_uint2(out[0] | (out[1] << 16), out[2] | (out[3] << 16));
    }
}

// fp16(q scale). Rounding up to the format's grid can pass the largest half; saturate: it does so for some value.
__device__ __forceinline__ uint32_t scaled_pair(uint32_t pair, float scale, bool saturate) {
    float2 x = __fmul2_rn(__half22float2(as_half2(pair)), make_float2(scale, scale));
    if (saturate) {
        x.x = x.x > 65504.0f ? 65504.0f : x.x < -65504.0f ? -65504.0f : x.x;
        x.y = x.y > 65504.0f ? 65504.0f : x.y < -65504.0f ? -65504.0f : x.y;
    }
    return pack_half2(x.x, x.y);
}

template <int kFormat>
__device__ __forceinline__ uint4 decode_vector(const uint2 bytes, float scale) {
    const uint2 a = widen4<kFormat>(bytes.x), b = widen4<kFormat>(bytes.y);
    const bool saturate = !(scale * (kFormat == KV_INT8 ? 128.0f : kFormat == KV_E4M3 ? 448.0f : 57344.0f) <= 65504.0f);
    return make_uint4(scaled_pair(a.x, scale, saturate), scaled_pair(a.y, scale, saturate), scaled_pair(b.x, scale, saturate),
                      scaled_pair(b.y, scale, saturate));
}

struct Geometry {
    uint32_t lanes_log2;         // lanes of a vector: the power of two at or above dim / 8
    uint32_t tokens_log2;        // tokens of a block's round; its other vectors are heads
    Divider by_token_tiles, by_head_tiles;
};

// kRounds: vectors of a thread, kRounds groups of tokens of the block.
template <int kFormat, bool kWrite, int kRounds>
__global__ void __launch_bounds__(kThreads) kv_copy_kernel(const __grid_constant__ KvCopyLaunch p, const __grid_constant__ Geometry geometry) {
    wait_for_prior_kernels_then_release_next();
    const uint32_t lane = threadIdx.x & ((1u << geometry.lanes_log2) - 1u), vector = threadIdx.x >> geometry.lanes_log2;
    uint32_t token_tile, head_tile;
    const uint32_t row = geometry.by_head_tiles.quotient(geometry.by_token_tiles.quotient(blockIdx.x, token_tile), head_tile);
    const uint32_t round_tokens = 1u << geometry.tokens_log2;
    const uint32_t block_heads = (kThreads >> geometry.lanes_log2) >> geometry.tokens_log2;
    const uint32_t first_token = token_tile * (kRounds * round_tokens) + (vector & (round_tokens - 1u));
    const uint32_t head = head_tile * block_heads + (vector >> geometry.tokens_log2);
    const bool live = lane * 8u < p.dim && head < p.heads;

    const int64_t first = (p.positions != nullptr ? __ldg(p.positions + row) : static_cast<int64_t>(p.start)) + first_token;
    const int64_t count = p.counts != nullptr ? __ldg(p.counts + row) : static_cast<int64_t>(p.tokens);
    constexpr int64_t kWidth = kFormat == KV_F16 ? 2 : 1;
    const uint32_t slot = p.first_slot + row;
    const int64_t outside = row * p.row_stride + first_token * p.token_stride + head * p.head_stride + lane * 8u;
    const int64_t inside = slot * p.cache.slot_stride + first * p.cache.token_stride + head * p.cache.head_stride + lane * 8u * kWidth;
    const int64_t scale_at = (static_cast<int64_t>(slot) * p.heads + head) * p.cache.capacity + first;
    bool exists[kRounds], present[kRounds];
#pragma unroll
    for (int i = 0; i < kRounds; ++i) {
        const uint32_t token = first_token + i * round_tokens;
        exists[i] = live && token < p.tokens;
        const int64_t at = first + i * static_cast<int64_t>(round_tokens);
        present[i] = exists[i] && token < count && at >= 0 && at < p.cache.capacity;
    }
    const int64_t outside_step = static_cast<int64_t>(round_tokens) * p.token_stride, inside_step = round_tokens * p.cache.token_stride;

    if constexpr (kWrite) {
        uint4 k[kRounds], v[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            k[i] = v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (present[i]) {
                k[i] = __ldcs(reinterpret_cast<const uint4*>(p.k + outside + i * outside_step));
                v[i] = __ldcs(reinterpret_cast<const uint4*>(p.v + outside + i * outside_step));
            }
        }
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            const int64_t to = inside + i * inside_step;
            if constexpr (kFormat == KV_F16) {
                if (present[i]) {
                    *reinterpret_cast<uint4*>(p.cache.k + to) = k[i];
                    *reinterpret_cast<uint4*>(p.cache.v + to) = v[i];
                }
            } else {
                float k_max = largest_finite(k[i]), v_max = largest_finite(v[i]);
                for (uint32_t offset = 1; offset < (1u << geometry.lanes_log2); offset <<= 1) {
                    k_max = fmaxf(k_max, __shfl_xor_sync(0xffffffffu, k_max, offset));
                    v_max = fmaxf(v_max, __shfl_xor_sync(0xffffffffu, v_max, offset));
                }
                const float2 k_scale = scale_of<kFormat>(k_max), v_scale = scale_of<kFormat>(v_max);
                if (present[i]) {
                    *reinterpret_cast<uint2*>(p.cache.k + to) = encode_vector<kFormat>(k[i], k_scale);
                    *reinterpret_cast<uint2*>(p.cache.v + to) = encode_vector<kFormat>(v[i], v_scale);
                    if (lane == 0) {
                        p.cache.k_scales[scale_at + i * round_tokens] = k_scale.x;
                        p.cache.v_scales[scale_at + i * round_tokens] = v_scale.x;
                    }
                }
            }
        }
    } else if constexpr (kFormat == KV_F16) {
        uint4 k[kRounds], v[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            k[i] = v[i] = make_uint4(0u, 0u, 0u, 0u);
            if (present[i]) {
                k[i] = __ldg(reinterpret_cast<const uint4*>(p.cache.k + inside + i * inside_step));
                v[i] = __ldg(reinterpret_cast<const uint4*>(p.cache.v + inside + i * inside_step));
            }
        }
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            if (!exists[i]) continue;
            *reinterpret_cast<uint4*>(p.k + outside + i * outside_step) = k[i];
            *reinterpret_cast<uint4*>(p.v + outside + i * outside_step) = v[i];
        }
    } else {
        uint2 k[kRounds], v[kRounds];
        float k_scale[kRounds], v_scale[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            k[i] = v[i] = make_uint2(0u, 0u);
            k_scale[i] = v_scale[i] = 1.0f;
            if (present[i]) {
                k[i] = __ldg(reinterpret_cast<const uint2*>(p.cache.k + inside + i * inside_step));
                v[i] = __ldg(reinterpret_cast<const uint2*>(p.cache.v + inside + i * inside_step));
                k_scale[i] = __ldg(p.cache.k_scales + scale_at + i * round_tokens);
                v_scale[i] = __ldg(p.cache.v_scales + scale_at + i * round_tokens);
            }
        }
#pragma unroll
        for (int i = 0; i < kRounds; ++i) {
            if (!exists[i]) continue;
            *reinterpret_cast<uint4*>(p.k + outside + i * outside_step) = decode_vector<kFormat>(k[i], k_scale[i]);
            *reinterpret_cast<uint4*>(p.v + outside + i * outside_step) = decode_vector<kFormat>(v[i], v_scale[i]);
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
    // long copies have two vectors of K and of V in flight per thread
    const uint32_t rounds = launch.tokens >= 8 * tokens ? 2u : 1u;
    const uint32_t token_tiles = (launch.tokens + rounds * tokens - 1) / (rounds * tokens), head_tiles = (launch.heads + heads - 1) / heads;
    const uint64_t blocks = static_cast<uint64_t>(token_tiles) * head_tiles * launch.rows;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    geometry.by_token_tiles.set(token_tiles);
    geometry.by_head_tiles.set(head_tiles);
    const auto run = [&](auto kernel) { return launch_behind(kernel, static_cast<uint32_t>(blocks), kThreads, 0, stream, early_launch, launch, geometry); };
    const auto run_format = [&](auto format) {
        constexpr int kFormat = decltype(format)::value;
        return rounds == 2 ? run(kv_copy_kernel<kFormat, kWrite, 2>) : run(kv_copy_kernel<kFormat, kWrite, 1>);
    };
    switch (launch.format) {
    case KV_E4M3: return run_format(std::integral_constant<int, KV_E4M3>{});
    case KV_E5M2: return run_format(std::integral_constant<int, KV_E5M2>{});
    case KV_INT8: return run_format(std::integral_constant<int, KV_INT8>{});
    default: return run_format(std::integral_constant<int, KV_F16>{});
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
