// Attention of few query rows per key head over long keys: tokens of sequences that share a prefix (see attention.cuh for
// rows, passes and blocks), and the kernel that joins the shares of the keys.
//
//   s_j = scale * q . k_j,  y = sum_j 2^(s_j log2 e - m) v_j / sum_j 2^(s_j log2 e - m)
// in one pass over the keys with a running m. The sums stay as they are when m grows by less than 2^7: weights are kept
// as halves, up to 2^6 at m and 2^13 above it, so that the smallest that a half resolves is 2^-31 of the weight at m.
//
// What bounds it: the bytes of the cache for long keys; for short ones latency, the start of a block and the first round trip to
// memory (256 keys for each of 64 sequences, 20 heads of 64 in FP16: 84 MB of cache room, of which 36 MB come from memory, in 19 us,
// caches cold). Every warp of a block takes every fourth group of 16 (FP16) or 32 (8-bit) keys
// and keeps its own sums, so that no warp waits for another before the end; keys and values go from global memory to the
// registers of the warp's MMAs, 4 KB (heads of 64) or 8 KB (128) of them in flight per warp, and through no shared
// memory. That works because the products do not care about the order of what they sum over:
//   S = Q K^T: lane (g = lane / 4, t = lane % 4) holds for key g of a group of eight 16 consecutive bytes of the head, so
//   the k index of the m16n8k16 MMA is a permutation of the head's dimensions, the same for Q.
//   O = P V: the lane holds for keys 2t, 2t + 1, 2t + 8, 2t + 9 eight consecutive dimensions 8g .. 8g + 7, and MMA j takes
//   the j-th of them, so its column g is dimension 8g + j.
// An 8-bit cache enters the MMAs as exact halves without its scales. A key's scale multiplies its column of S; a value's
// multiplies its weight, and the halves hold that product relative to the largest so far of the keys that the row sees: O is kept
// divided by 2^lift, lift the largest of s_j log2 e - m + log2(value scale), which like m moves by more than 2^7 only.

#include "attention.cuh"

namespace sdxlq {

namespace {

constexpr uint32_t kWarps = 4;
constexpr float kWeightBits = 6.0f;      // a weight at the running maximum is 2^6
constexpr float kSlackBits = 7.0f;       // the maximum may be passed by this much before the sums are rescaled

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_vector16(const uint8_t* base, bool inside) {
    return inside ? __ldg(reinterpret_cast<const uint4*>(base)) : make_uint4(0u, 0u, 0u, 0u);
}
__device__ __forceinline__ uint2 load_vector8(const uint8_t* base, bool inside) {
    return inside ? __ldg(reinterpret_cast<const uint2*>(base)) : make_uint2(0u, 0u);
}

// A group of keys in registers, as the MMAs take it.
template <int kDim, int kFormat>
struct KeyBlock {
    static constexpr bool kHalf = kFormat == KV_F16;
    static constexpr int kKeys = kHalf ? 16 : 32;
    static constexpr int kTiles = kKeys / 8;             // groups of eight keys
    static constexpr int kVectors = kHalf ? kDim / 32 : kDim / 64;
    uint4 word[kTiles][kVectors];
    float scale[kHalf ? 1 : kTiles][2];

    __device__ __forceinline__ void load(const KvView& view, const uint8_t* keys, const float* scales, uint32_t first, uint32_t end,
                                         uint32_t dim, uint32_t g, uint32_t t) {
#pragma unroll
        for (int tile = 0; tile < kTiles; ++tile) {
            const uint32_t key = first + tile * 8u + g;
            const uint8_t* const row = keys + key * view.token_stride;
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                const uint32_t d = kHalf ? v * 32u + t * 8u : v * 64u + t * 16u;
                word[tile][v] = load_vector16(row + d * (kHalf ? 2u : 1u), key < end && d < dim);
            }
            if constexpr (!kHalf) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t column = first + tile * 8u + 2u * t + i;
                    scale[tile][i] = column < end ? __ldg(scales + column) : 0.0f;
                }
            }
        }
    }

    // The B operand of MMA step `step` (16 dimensions) for group `tile`.
    __device__ __forceinline__ uint2 operand(int tile, int step) const {
        if constexpr (kHalf) {
            const uint4 w = word[tile][step / 2];
            return step % 2 == 0 ? make_uint2(w.x, w.y) : make_uint2(w.z, w.w);
        } else {
            const uint4 w = word[tile][step / 4];
            const uint32_t bytes = step % 4 == 0 ? w.x : step % 4 == 1 ? w.y : step % 4 == 2 ? w.z : w.w;
            return widen4<kFormat>(bytes);
        }
    }

    // First of the four dimensions that lane t has in MMA step `step`.
    static __device__ __forceinline__ uint32_t dimension(int step, uint32_t t) {
        return kHalf ? step / 2 * 32u + t * 8u + step % 2 * 4u : step / 4 * 64u + t * 16u + step % 4 * 4u;
    }
};

template <int kDim, int kFormat>
struct ValueBlock {
    static constexpr bool kHalf = kFormat == KV_F16;
    static constexpr int kKeys = kHalf ? 16 : 32;
    static constexpr int kVectors = kDim / 64;
    uint4 word16[kHalf ? kKeys / 4 : 1][kVectors];
    uint2 word8[kHalf ? 1 : kKeys / 4][kVectors];
    float scale[kHalf ? 1 : kKeys / 4];

    // the lane's i-th key of the group
    static __device__ __forceinline__ uint32_t key_of(int i, uint32_t t) { return i / 4 * 16u + i / 2 % 2 * 8u + 2u * t + i % 2; }

    __device__ __forceinline__ void load(const KvView& view, const uint8_t* values, const float* scales, uint32_t first, uint32_t end,
                                         uint32_t dim, uint32_t g, uint32_t t) {
#pragma unroll
        for (int i = 0; i < kKeys / 4; ++i) {
            const uint32_t key = first + key_of(i, t);
            const uint8_t* const row = values + key * view.token_stride;
#pragma unroll
            for (int v = 0; v < kVectors; ++v) {
                const uint32_t d = v * 64u + g * 8u;
                if constexpr (kHalf) word16[i][v] = load_vector16(row + d * 2u, key < end && d < dim);
                else word8[i][v] = load_vector8(row + d, key < end && d < dim);
            }
            if constexpr (!kHalf) scale[i] = key < end ? __ldg(scales + key) : 0.0f;
        }
    }

    // A vector of zeros adds nothing whatever its scale is (1, where the cache was written from zeros), and must not be what the
    // other weights are placed by: its scale becomes 0. Every eight lanes of a key have a part of it; the groups' 32 keys make
    // the bits of one word.
    __device__ __forceinline__ void drop_zero_vectors(uint32_t t) {
        static_assert(kKeys == 32);
        uint32_t lives = 0;
#pragma unroll
        for (int i = 0; i < kKeys / 4; ++i) {
            uint32_t bits = 0;
#pragma unroll
            for (int v = 0; v < kVectors; ++v) bits |= word8[i][v].x | word8[i][v].y;
            if ((bits & magnitude_bits<kFormat>()) != 0) lives |= 1u << i;
        }
        lives = __reduce_or_sync(0xffffffffu, lives << (8u * t)) >> (8u * t);
#pragma unroll
        for (int i = 0; i < kKeys / 4; ++i) {
            if ((lives >> i & 1u) == 0) scale[i] = 0.0f;
        }
    }

    // The B operands of the 16 keys `step` for dimensions 4 `quad` .. + 3 of the lane's eight in vector v: four MMAs.
    __device__ __forceinline__ void operands(int step, int v, int quad, uint32_t (&b0)[4], uint32_t (&b1)[4]) const {
        if constexpr (kHalf) {
#pragma unroll
            for (int pair = 0; pair < 2; ++pair) {
                uint32_t w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint4 x = word16[step * 4 + i][v];
                    w[i] = quad == 0 ? (pair == 0 ? x.x : x.y) : (pair == 0 ? x.z : x.w);
                }
                b0[pair * 2] = __byte_perm(w[0], w[1], 0x5410);
                b0[pair * 2 + 1] = __byte_perm(w[0], w[1], 0x7632);
                b1[pair * 2] = __byte_perm(w[2], w[3], 0x5410);
                b1[pair * 2 + 1] = __byte_perm(w[2], w[3], 0x7632);
            }
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = quad == 0 ? word8[step * 4 + i][v].x : word8[step * 4 + i][v].y;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const uint32_t select = half == 0 ? 0x5140u : 0x7362u;
                const uint2 a = widen4<kFormat>(__byte_perm(w[0], w[1], select)), b = widen4<kFormat>(__byte_perm(w[2], w[3], select));
                b0[half * 2] = a.x;
                b0[half * 2 + 1] = a.y;
                b1[half * 2] = b.x;
                b1[half * 2 + 1] = b.y;
            }
        }
    }
};

__device__ __forceinline__ bool has_non_finite(uint32_t pair) {
    return (pair & 0x7C00u) == 0x7C00u || (pair & 0x7C000000u) == 0x7C000000u;
}

// kRowTiles: tiles of 16 rows per warp.
template <int kDim, int kFormat, int kRowTiles>
__global__ void __launch_bounds__(32 * kWarps) attention_rows_kernel(const __grid_constant__ AttentionParams p) {
    using Keys = KeyBlock<kDim, kFormat>;
    using Values = ValueBlock<kDim, kFormat>;
    constexpr int kSteps = kDim / 16, kKeys = Keys::kKeys, kTiles = Keys::kTiles;
    constexpr int kTileRows = 16 * kRowTiles, kPitch = kDim + 4;
    constexpr bool kScaled = kFormat != KV_F16;
    extern __shared__ float shared[];
    float* const shared_o = shared;                                      // [kWarps][kTileRows][kPitch]
    float* const shared_m = shared + kWarps * kTileRows * kPitch;        // [kWarps][kTileRows]
    float* const shared_l = shared_m + kWarps * kTileRows;

    wait_for_prior_kernels_then_release_next();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const BlockPlace here = place_block(p, blockIdx.x);
    const AttentionPass& pass = p.pass[here.pass];
    const uint32_t kv_head = here.kv_head, first_member = here.first_member, first_row = here.row_tile * kTileRows;

    // the keys of the block: blocks of the prefix, then of the entry's own keys
    const uint32_t prefix_slot = pass.with_prefix ? p.by_rows_per_prefix.quotient(first_member) : 0u;
    const uint32_t prefix_length = pass.with_prefix ? length_of(p.prefix, prefix_slot) : 0u;
    const uint32_t own_length = pass.with_own ? length_of(p.own, first_member) : 0u;
    const uint32_t last_row = min(first_row + kTileRows, pass.rows) - 1u;        // sees the most of its entry's own keys
    const uint32_t own_seen = p.causal && pass.with_own ? causal_limit(own_length, p.q_tokens, p.by_repeat.quotient(last_row)) : own_length;
    const uint32_t prefix_blocks = (prefix_length + kKeys - 1) / kKeys, own_blocks = (own_seen + kKeys - 1) / kKeys;
    const uint64_t blocks = static_cast<uint64_t>(prefix_blocks) + own_blocks;
    const uint32_t block_begin = static_cast<uint32_t>(blocks * here.split / pass.splits);
    const uint32_t block_end = static_cast<uint32_t>(blocks * (here.split + 1) / pass.splits);

    // Q, and how many own keys each of the lane's rows sees
    uint32_t q[kRowTiles][kSteps][4];
    uint32_t limit[kRowTiles][2];
    uint32_t least_limit = own_length;
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t r = first_row + rt * 16u + half * 8u + g;
            const bool inside = r < pass.rows;
            const QueryRow at = locate_row(p, first_member, kv_head, inside ? r : 0u);
            const __half* const row = p.q + at.batch * p.q_batch + at.token * p.q_token + at.head * p.q_head;
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                const uint32_t d = Keys::dimension(step, t);
                const uint2 x = inside && d < p.dim ? __ldg(reinterpret_cast<const uint2*>(row + d)) : make_uint2(0u, 0u);
                q[rt][step][half] = x.x;
                q[rt][step][half + 2] = x.y;
            }
            limit[rt][half] = p.causal ? causal_limit(own_length, p.q_tokens, at.token) : own_length;
            least_limit = min(least_limit, limit[rt][half]);
        }
    }
    least_limit = __reduce_min_sync(0xffffffffu, least_limit);

    float o[kRowTiles][kDim / 8][4] = {};
    float row_max[kRowTiles][2], row_sum[kRowTiles][2];
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt) {
        row_max[rt][0] = row_max[rt][1] = __int_as_float(0xff800000);
        row_sum[rt][0] = row_sum[rt][1] = 0.0f;
    }
    float lift[kScaled ? kRowTiles : 1][2];       // 8-bit caches: O is relative to 2^lift; nothing seen yet is far below any
#pragma unroll
    for (int rt = 0; rt < (kScaled ? kRowTiles : 1); ++rt) lift[rt][0] = lift[rt][1] = -1000.0f;

    const auto rescale = [&](int rt, float factor0, float factor1) {
#pragma unroll
        for (int n = 0; n < kDim / 8; ++n) {
            o[rt][n][0] *= factor0;
            o[rt][n][1] *= factor0;
            o[rt][n][2] *= factor1;
            o[rt][n][3] *= factor1;
        }
    };

    // where a block's keys are
    struct Place {
        const uint8_t* k;
        const uint8_t* v;
        const float* k_scales;
        const float* v_scales;
        uint32_t first, end;
    };
    const auto view_of = [&](uint32_t block) -> const KvView& { return block < prefix_blocks ? p.prefix : p.own; };
    const auto place = [&](uint32_t block) {
        const bool in_prefix = block < prefix_blocks;
        const KvView& view = view_of(block);
        const int64_t slot = in_prefix ? prefix_slot : first_member;
        const int64_t base = slot * view.slot_stride + kv_head * view.head_stride;
        const int64_t scales = (slot * p.kv_heads + kv_head) * view.capacity;
        Place at;
        at.k = view.k + base;
        at.v = view.v + base;
        at.k_scales = kScaled ? view.k_scales + scales : nullptr;
        at.v_scales = kScaled ? view.v_scales + scales : nullptr;
        at.first = (in_prefix ? block : block - prefix_blocks) * kKeys;
        at.end = in_prefix ? prefix_length : own_length;
        return at;
    };

    Keys keys;
    Values values;
    uint32_t block = block_begin + warp;
    if (block < block_end) {
        const Place at = place(block);
        keys.load(view_of(block), at.k, at.k_scales, at.first, at.end, p.dim, g, t);
        values.load(view_of(block), at.v, at.v_scales, at.first, at.end, p.dim, g, t);
    }
    while (block < block_end) {
        const bool in_prefix = block < prefix_blocks;
        const uint32_t first = (in_prefix ? block : block - prefix_blocks) * kKeys;
        const uint32_t next = block + kWarps;

        float s[kRowTiles][kTiles][4] = {};
#pragma unroll
        for (int tile = 0; tile < kTiles; ++tile) {
#pragma unroll
            for (int step = 0; step < kSteps; ++step) {
                const uint2 b = keys.operand(tile, step);
#pragma unroll
                for (int rt = 0; rt < kRowTiles; ++rt) mma_f16(s[rt][tile], q[rt][step], b.x, b.y);
            }
        }
        float key_scale[kTiles][2];
        if constexpr (kScaled) {
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                key_scale[tile][0] = keys.scale[tile][0] * p.scale_log2;
                key_scale[tile][1] = keys.scale[tile][1] * p.scale_log2;
            }
        }
        if (next < block_end) {          // the next keys travel while this block is worked on
            const Place at = place(next);
            keys.load(view_of(next), at.k, at.k_scales, at.first, at.end, p.dim, g, t);
        }

        const uint32_t seen_by_all = in_prefix ? prefix_length : least_limit;
        const bool masked = first + kKeys > seen_by_all;
        float bits[kScaled ? kKeys / 4 : 1];
        if constexpr (kScaled) {
            values.drop_zero_vectors(t);
#pragma unroll
            for (int i = 0; i < kKeys / 4; ++i) bits[i] = place_bits(values.scale[i]);
        }

        uint32_t weights[kRowTiles][kTiles / 2][4];
#pragma unroll
        for (int rt = 0; rt < kRowTiles; ++rt) {
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s[rt][tile][c] *= kScaled ? key_scale[tile][c & 1] : p.scale_log2;
                    if (masked) {
                        const uint32_t key = first + tile * 8u + 2u * t + (c & 1);
                        if (key >= (in_prefix ? prefix_length : limit[rt][c >> 1])) s[rt][tile][c] = __int_as_float(0xff800000);
                    }
                }
            }
            // Differences of scores, not sums with the reference, decide and make the weights: they are exact for neighbours of any size.
            float grow[2], lower[2];                                     // of the row's sum, and of O
            bool grown = false;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float largest = __int_as_float(0xff800000);
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) largest = fmaxf(largest, fmaxf(s[rt][tile][2 * half], s[rt][tile][2 * half + 1]));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
                const float over = largest - row_max[rt][half];          // NaN where neither is there
                const bool moves = over > kSlackBits;
                if (moves) row_max[rt][half] = largest;
                grown = grown || moves;
                grow[half] = lower[half] = moves ? exp2_approx(-over) : 1.0f;
                const float reference = row_max[rt][half] > __int_as_float(0xff800000) ? row_max[rt][half] : 0.0f;
                float above = __int_as_float(0xff800000);
#pragma unroll
                for (int tile = 0; tile < kTiles; ++tile) {
#pragma unroll
                    for (int c = 2 * half; c < 2 * half + 2; ++c) {
                        s[rt][tile][c] -= reference;
                        if constexpr (kScaled) above = fmaxf(above, s[rt][tile][c] + bits[tile / 2 * 4 + tile % 2 * 2 + (c & 1)]);
                    }
                }
                if constexpr (kScaled) {
                    above = fmaxf(above, __shfl_xor_sync(0xffffffffu, above, 1));
                    above = fmaxf(above, __shfl_xor_sync(0xffffffffu, above, 2));
                    const float kept = moves ? lift[rt][half] - over : lift[rt][half];
                    if (moves || above > kept + kSlackBits) {
                        lift[rt][half] = fmaxf(kept, above);
                        lower[half] = exp2_approx(kept - lift[rt][half]);
                        grown = true;
                    }
                }
            }
            if (__any_sync(0xffffffffu, grown)) {
                row_sum[rt][0] *= grow[0];
                row_sum[rt][1] *= grow[1];
                rescale(rt, lower[0], lower[1]);
            }
            float unit[2] = {1.0f, 1.0f};                                // 2^(-lift / 2): a lift may be as large as the largest scale's
            if constexpr (kScaled) {
                unit[0] = exp2_approx(-0.5f * lift[rt][0]);
                unit[1] = exp2_approx(-0.5f * lift[rt][1]);
            }
#pragma unroll
            for (int tile = 0; tile < kTiles; ++tile) {
                float w[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    w[c] = exp2_approx(s[rt][tile][c] + kWeightBits);
                    row_sum[rt][c >> 1] += w[c];
                    if constexpr (kScaled) {
                        const float factor = values.scale[tile / 2 * 4 + tile % 2 * 2 + (c & 1)] * unit[c >> 1] * unit[c >> 1];
                        w[c] = s[rt][tile][c] == __int_as_float(0xff800000) ? 0.0f : w[c] * factor;
                    }
                }
                weights[rt][tile / 2][tile % 2 * 2] = pack_half2(w[0], w[1]);
                weights[rt][tile / 2][tile % 2 * 2 + 1] = pack_half2(w[2], w[3]);
            }
        }

        // A value that is not finite makes 0 * v a NaN, also where the weight is 0 because the row does not see the key.
        // Keys behind a sequence's end were loaded as zeros; those that the causal mask hides from some rows of the tile
        // and not from others are looked through here.
        bool row_by_row = false;
        if (kFormat != KV_INT8 && masked && !in_prefix && p.causal) {
            bool found = false;
#pragma unroll
            for (int step = 0; step < kKeys / 16; ++step) {
#pragma unroll
                for (int v = 0; v < Values::kVectors; ++v) {
#pragma unroll
                    for (int quad = 0; quad < 2; ++quad) {
                        uint32_t b0[4], b1[4];
                        values.operands(step, v, quad, b0, b1);
#pragma unroll
                        for (int i = 0; i < 4; ++i) found = found || has_non_finite(b0[i]) || has_non_finite(b1[i]);
                    }
                }
            }
            row_by_row = __any_sync(0xffffffffu, found);
        }
        if (!row_by_row) {
#pragma unroll
            for (int step = 0; step < kKeys / 16; ++step) {
#pragma unroll
                for (int v = 0; v < Values::kVectors; ++v) {
#pragma unroll
                    for (int quad = 0; quad < 2; ++quad) {
                        uint32_t b0[4], b1[4];
                        values.operands(step, v, quad, b0, b1);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
#pragma unroll
                            for (int rt = 0; rt < kRowTiles; ++rt) mma_f16(o[rt][v * 8 + quad * 4 + i], weights[rt][step], b0[i], b1[i]);
                        }
                    }
                }
            }
        } else {
            // one row at a time, the keys that it does not see as zeros
            for (int rt = 0; rt < kRowTiles; ++rt) {
                for (uint32_t r = 0; r < 16; ++r) {
                    const uint32_t mine = r < 8 ? limit[0][0] : limit[0][1];
                    const uint32_t other = kRowTiles > 1 ? (r < 8 ? limit[kRowTiles - 1][0] : limit[kRowTiles - 1][1]) : mine;
                    const uint32_t seen = __shfl_sync(0xffffffffu, rt == 0 ? mine : other, (r & 7u) * 4u);
#pragma unroll
                    for (int step = 0; step < kKeys / 16; ++step) {
                        const uint32_t key = first + step * 16u + 2u * t;
                        const uint32_t keep0 = (key < seen ? 0xFFFFu : 0u) | (key + 1u < seen ? 0xFFFF0000u : 0u);
                        const uint32_t keep1 = (key + 8u < seen ? 0xFFFFu : 0u) | (key + 9u < seen ? 0xFFFF0000u : 0u);
#pragma unroll
                        for (int v = 0; v < Values::kVectors; ++v) {
#pragma unroll
                            for (int quad = 0; quad < 2; ++quad) {
                                uint32_t b0[4], b1[4];
                                values.operands(step, v, quad, b0, b1);
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const int n = v * 8 + quad * 4 + i;
#pragma unroll
                                    for (int tile = 0; tile < kRowTiles; ++tile) {
                                        float sum[4] = {};
                                        mma_f16(sum, weights[tile][step], b0[i] & keep0, b1[i] & keep1);
                                        if (tile == rt && g == (r & 7u)) {
                                            if (r < 8) {
                                                o[tile][n][0] += sum[0];
                                                o[tile][n][1] += sum[1];
                                            } else {
                                                o[tile][n][2] += sum[2];
                                                o[tile][n][3] += sum[3];
                                            }
                                        }
                                    }
                                }
                            }
                        }
                    }
                }
            }
        }
        if (next < block_end) {
            const Place at = place(next);
            values.load(view_of(next), at.v, at.v_scales, at.first, at.end, p.dim, g, t);
        }
        block = next;
    }

    // the warps' sums meet in shared memory
#pragma unroll
    for (int rt = 0; rt < kRowTiles; ++rt) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            float sum = row_sum[rt][half];
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            const uint32_t r = rt * 16u + half * 8u + g;
            if (t == 0) {
                shared_m[warp * kTileRows + r] = row_max[rt][half];
                shared_l[warp * kTileRows + r] = sum;
            }
            float* const row = shared_o + (warp * kTileRows + r) * kPitch;
            const float unit = kScaled ? exp2_approx(0.5f * lift[kScaled ? rt : 0][half]) : 1.0f;
#pragma unroll
            for (int v = 0; v < kDim / 64; ++v) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    row[v * 64 + 16u * t + j] = o[rt][v * 8 + j][2 * half] * unit * unit;
                    row[v * 64 + 16u * t + 8 + j] = o[rt][v * 8 + j][2 * half + 1] * unit * unit;
                }
            }
        }
    }
    __syncthreads();
    for (uint32_t index = threadIdx.x; index < kTileRows * (kDim / 8); index += 32 * kWarps) {
        const uint32_t r = index / (kDim / 8), d = index % (kDim / 8) * 8u;
        if (first_row + r >= pass.rows || d >= p.dim) continue;
        float largest = __int_as_float(0xff800000);
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) largest = fmaxf(largest, shared_m[w * kTileRows + r]);
        float total = 0.0f, sum[8] = {};
        if (largest > __int_as_float(0xff800000)) {
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                const float share = exp2_approx(shared_m[w * kTileRows + r] - largest);
                total = fmaf(shared_l[w * kTileRows + r], share, total);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] = fmaf(shared_o[(w * kTileRows + r) * kPitch + d + j], share, sum[j]);
            }
        } else {
            // no score above -inf: an empty row, or one whose scores are all NaN or -inf, which carries its sums' NaN
#pragma unroll
            for (uint32_t w = 0; w < kWarps; ++w) {
                total += shared_l[w * kTileRows + r];
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] += shared_o[(w * kTileRows + r) * kPitch + d + j];
            }
        }
        const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
        const QueryRow at = locate_row(p, first_member, kv_head, first_row + r);
        if (writes_output(p, here)) {
            __half* const row = p.y + at.batch * p.y_batch + at.token * p.y_token + at.head * p.y_head + d;
            const uint4 packed = make_uint4(pack_half2(sum[0] * inverse, sum[1] * inverse), pack_half2(sum[2] * inverse, sum[3] * inverse),
                                            pack_half2(sum[4] * inverse, sum[5] * inverse), pack_half2(sum[6] * inverse, sum[7] * inverse));
            *reinterpret_cast<uint4*>(row) = packed;
        } else {
            const uint64_t row = (static_cast<uint64_t>(at.batch) * p.q_tokens + at.token) * p.q_heads + at.head;
            const uint64_t place_in_slot = scratch_row(p, here, kTileRows, r, row);
            float4* const out = reinterpret_cast<float4*>(p.part_o + place_in_slot * p.dim + d);
            out[0] = make_float4(sum[0] * inverse, sum[1] * inverse, sum[2] * inverse, sum[3] * inverse);
            out[1] = make_float4(sum[4] * inverse, sum[5] * inverse, sum[6] * inverse, sum[7] * inverse);
            if (d == 0) {
                const float kNone = __int_as_float(0xff800000);
                p.part_lse[place_in_slot] = make_float2(total == 0.0f ? kNone : largest > kNone ? largest : 0.0f, log2f(total) - kWeightBits);
            }
        }
    }
}

// y = sum_s 2^lse_s o_s / sum_s 2^lse_s over the shares of each row. A warp takes a row: its lanes find the largest lse, then
// take eight dimensions each of every 256 / dim-th share, which meet in lane order. What bounds it: latency, two round trips to
// the L2 cache, which holds the shares; with a lane per row and eight dimensions that walked over the shares one by one it
// took 24 us for 1280 rows of 30 shares.
constexpr uint32_t kJoinWarps = 4;

__global__ void __launch_bounds__(32 * kJoinWarps) attention_join_kernel(const __grid_constant__ AttentionParams p, uint32_t pass_index, uint32_t tile_rows) {
    wait_for_prior_kernels_then_release_next();
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t rows = p.slot_rows, row = static_cast<uint64_t>(blockIdx.x) * kJoinWarps + (threadIdx.x >> 5);
    if (row >= rows) return;
    uint64_t b, token;
    uint32_t head;
    if (p.by_row) {
        const uint64_t position = row / p.q_heads;
        head = static_cast<uint32_t>(row % p.q_heads);
        b = position / p.q_tokens;
        token = position % p.q_tokens;
    } else {
        const BlockPlace tile = place_block(p, (pass_index ? p.pass[0].tiles * p.pass[0].splits : 0u) + static_cast<uint32_t>(row / tile_rows));
        const uint32_t r = tile.row_tile * tile_rows + static_cast<uint32_t>(row % tile_rows);
        if (r >= p.pass[pass_index].rows) return;
        const QueryRow at = locate_row(p, tile.first_member, tile.kv_head, r);
        b = at.batch;
        token = at.token;
        head = at.head;
    }
    const float kNone = __int_as_float(0xff800000);
    float2 largest = make_float2(kNone, 0.0f);
    for (uint32_t s = lane; s < p.slots; s += 32) {
        const float2 lse = __ldg(p.part_lse + s * rows + row);
        if ((lse.x - largest.x) + (lse.y - largest.y) > 0.0f) largest = lse;
    }
#pragma unroll
    for (int offset = 16; offset != 0; offset >>= 1) {
        const float2 other = make_float2(__shfl_xor_sync(0xffffffffu, largest.x, offset), __shfl_xor_sync(0xffffffffu, largest.y, offset));
        const float ahead = (other.x - largest.x) + (other.y - largest.y);
        // one answer for both lanes of the pair, also where the two are equal in sum and not in their parts
        if (ahead > 0.0f || (ahead == 0.0f && other.x > largest.x)) largest = other;
    }
    const uint32_t lanes_log2 = p.dim > 64 ? 4u : 3u, d = (lane & ((1u << lanes_log2) - 1u)) * 8u, groups = 32u >> lanes_log2;
    float total = 0.0f, sum[8] = {};
    for (uint32_t s = lane >> lanes_log2; s < p.slots; s += groups) {
        const float2 lse = __ldg(p.part_lse + s * rows + row);
        const bool counts = lse.x != kNone;                      // else an empty share
        const float share = counts ? exp2_approx((lse.x - largest.x) + (lse.y - largest.y)) : 0.0f;
        total += share;
        if (counts && d < p.dim) {
            const float4* const part = reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * p.dim + d);
            const float4 x = __ldg(part), y = __ldg(part + 1);
            sum[0] = fmaf(x.x, share, sum[0]); sum[1] = fmaf(x.y, share, sum[1]); sum[2] = fmaf(x.z, share, sum[2]); sum[3] = fmaf(x.w, share, sum[3]);
            sum[4] = fmaf(y.x, share, sum[4]); sum[5] = fmaf(y.y, share, sum[5]); sum[6] = fmaf(y.z, share, sum[6]); sum[7] = fmaf(y.w, share, sum[7]);
        }
    }
    for (uint32_t offset = 16; offset >= (1u << lanes_log2); offset >>= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, offset);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], offset);
    }
    if (lane >> lanes_log2 != 0 || d >= p.dim) return;
    const float inverse = total == 0.0f ? 0.0f : 1.0f / total;
    __half* const out = p.y + b * p.y_batch + token * p.y_token + head * p.y_head + d;
    *reinterpret_cast<uint4*>(out) = make_uint4(pack_half2(sum[0] * inverse, sum[1] * inverse), pack_half2(sum[2] * inverse, sum[3] * inverse),
                                                pack_half2(sum[4] * inverse, sum[5] * inverse), pack_half2(sum[6] * inverse, sum[7] * inverse));
}

template <int kDim, int kFormat, int kRowTiles>
cudaError_t launch_tile(const AttentionParams& params, cudaStream_t stream, bool early_launch) {
    constexpr size_t bytes = sizeof(float) * kWarps * 16 * kRowTiles * (kDim + 4 + 2);
    auto* const kernel = attention_rows_kernel<kDim, kFormat, kRowTiles>;
    if constexpr (bytes > 48 * 1024) {
        const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
        if (error != cudaSuccess) return error;
    }
    uint32_t blocks = 0;
    for (uint32_t i = 0; i < params.pass_count; ++i) blocks += params.pass[i].tiles * params.pass[i].splits;
    return launch_behind(kernel, blocks, 32 * kWarps, bytes, stream, early_launch, params);
}

template <int kFormat>
cudaError_t launch_format(const AttentionParams& params, uint32_t row_tile, cudaStream_t stream, bool early_launch) {
    if (params.dim <= 64) {
        return row_tile == 16 ? launch_tile<64, kFormat, 1>(params, stream, early_launch) : launch_tile<64, kFormat, 2>(params, stream, early_launch);
    }
    return launch_tile<128, kFormat, 1>(params, stream, early_launch);       // two tiles of 128 dimensions are more than the registers hold
}

}  // namespace

cudaError_t launch_attention_rows(const AttentionParams& params, KvFormat format, uint32_t row_tile, cudaStream_t stream,
                                  bool early_launch) {
    switch (format) {
    case KV_E4M3: return launch_format<KV_E4M3>(params, row_tile, stream, early_launch);
    case KV_E5M2: return launch_format<KV_E5M2>(params, row_tile, stream, early_launch);
    case KV_INT8: return launch_format<KV_INT8>(params, row_tile, stream, early_launch);
    default: return launch_format<KV_F16>(params, row_tile, stream, early_launch);
    }
}

// Launched behind the others' end, not early: blocks of it that waited on the SMs cost the kernel before it 30 of 147 us in the
// self-attention of 2 x 4096 tokens.
cudaError_t launch_attention_join(const AttentionParams& params, uint32_t tile_rows, cudaStream_t stream) {
    const uint32_t pass = params.pass_count > 1 && params.pass[1].splits > 1 ? 1u : 0u;
    const uint64_t blocks = (params.slot_rows + kJoinWarps - 1) / kJoinWarps;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    return launch_behind(attention_join_kernel, static_cast<uint32_t>(blocks), 32 * kJoinWarps, 0, stream, false, params, pass, tile_rows);
}

}  // namespace sdxlq
