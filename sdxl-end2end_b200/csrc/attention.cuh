// Structures of the attention operators shared by the host dispatch and the kernels, and the arithmetic of a cache's
// 8-bit types.
#pragma once

#include "fp8_math.cuh"
#include "int8_math.cuh"
#include "quantize.cuh"

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

namespace sdxlq {

// Element type of a cache: the values of sdxlq_dtype.
enum KvFormat : int { KV_E4M3 = 0, KV_E5M2 = 1, KV_INT8 = 2, KV_F16 = 3 };

// Keys and values of some sequences. Strides in bytes.
struct KvView {
    uint8_t* k;
    uint8_t* v;
    float* k_scales;             // [slots, heads, capacity], null for FP16
    float* v_scales;
    const int32_t* lengths;      // [slots] or null: every slot holds `capacity` tokens (attention only)
    int64_t slot_stride, token_stride, head_stride;
    uint32_t slots, capacity;
};

// ---- writing and reading a cache ------------------------------------------------------------------------
struct KvCopyLaunch {
    KvView cache;
    __half* k;                   // FP16 tokens
    __half* v;
    int64_t row_stride, token_stride, head_stride;      // elements
    const int32_t* positions;    // [rows] or null: `start`
    const int32_t* counts;       // [rows] or null: all `tokens`
    uint32_t rows, tokens, heads, dim;
    uint32_t first_slot, start;
    uint32_t format;             // KvFormat
};
cudaError_t launch_kv_write(const KvCopyLaunch& launch, cudaStream_t stream, bool early_launch);
cudaError_t launch_kv_read(const KvCopyLaunch& launch, cudaStream_t stream, bool early_launch);

// ---- attention ------------------------------------------------------------------------------------------

// Division of n < 2^31 by a number known at the launch, as a multiplication (Granlund and Montgomery, PLDI 1994).
struct Divider {
    uint32_t divisor, magic, shift;
    void set(uint32_t d) {
        divisor = d;
        for (shift = 0; (uint64_t(1) << shift) < d; ++shift) {}
        magic = static_cast<uint32_t>((((uint64_t(1) << shift) - d) << 32) / d + 1);
    }
    __device__ __forceinline__ uint32_t quotient(uint32_t n) const { return (__umulhi(n, magic) + n) >> shift; }
    __device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t& rest) const {
        const uint32_t q = quotient(n);
        rest = n - q * divisor;
        return q;
    }
};

// Query rows of one key head are numbered r = (member * q_tokens + token) * repeat + head within the key head's group:
// rows of several batch entries that read the same keys stand behind one another.
//
// A launch runs one or two passes. A pass takes `members` batch entries together (all that share a prefix, or one) over
// the prefix, over the entries' own keys (members == 1), or over the one and then the other. Its tiles are tiles of rows of
// one key head, numbered (group, key head, row tile), and each of its blocks takes one of them over one of `splits` shares
// of the keys. Where a row gets its result from one block alone, that block writes it; else every block leaves its share in
// the scratch and the join kernel adds them up, either over all rows (the passes are the parts of every row: `by_row`), or
// over the tiles of one pass.
struct AttentionPass {
    uint32_t members, groups;    // batch = members * groups
    uint32_t rows;               // members * q_tokens * repeat
    uint32_t row_tiles, splits;
    uint32_t first_tile, tiles;  // of row_tiles * kv_heads * groups
    Divider by_tiles, by_row_tiles;
    uint32_t first_slot;         // by_row: scratch slot of split 0
    uint32_t with_prefix, with_own;
};
constexpr uint32_t kMaxPasses = 2;

struct AttentionParams {
    const __half* q;
    __half* y;
    int64_t q_batch, q_token, q_head;        // strides, elements
    int64_t y_batch, y_token, y_head;
    KvView prefix, own;
    uint32_t batch, q_tokens, q_heads, kv_heads, repeat, dim;
    uint32_t rows_per_prefix;    // batch entries that share a prefix
    Divider by_q_tokens, by_repeat, by_kv_heads, by_rows_per_prefix;
    uint32_t causal;
    float scale_log2;            // softmax scale * log2(e)
    uint32_t pass_count;
    AttentionPass pass[kMaxPasses];
    uint32_t by_row;
    uint32_t slots;              // shares of a row: all passes' splits, or those of the pass that has more than one
    uint64_t slot_rows;          // rows of a slot: batch * q_tokens * q_heads, or that pass's tiles * tile rows
    float* part_o;               // [slots, slot_rows, dim] shares, each divided by its own sum
    float2* part_lse;            // [slots, slot_rows] log2 of the sum of 2^score in two parts, which scores of
                                 // any size leave exact; -inf in the first for an empty share
};

cudaError_t launch_attention_rows(const AttentionParams& params, KvFormat format, uint32_t row_tile, cudaStream_t stream,
                                  bool early_launch);

constexpr uint32_t kTileKeys = 64;       // of a tile on the tensor memory
// Blocks of that kernel on an SM, by their tensor memory, shared memory and registers.
__host__ __device__ constexpr uint32_t tile_blocks_per_sm(uint32_t dim, KvFormat format) { return dim > 64 ? 2 : format == KV_F16 ? 4 : 3; }

// Tensor maps of FP16 keys and values, [slot, token, head, d], whose box is a tile of one head (64 of its dimensions).
struct AttentionMaps {
    CUtensorMap map[2][2];       // prefix, own; keys, values
};

cudaError_t launch_attention_tiles(const AttentionParams& params, const AttentionMaps& maps, KvFormat format, uint32_t* error_word,
                                   long long wait_limit_cycles, cudaStream_t stream, bool early_launch);
// tile_rows: of the pass that is joined (by_row: not used).
cudaError_t launch_attention_join(const AttentionParams& params, uint32_t tile_rows, cudaStream_t stream);

// A block's place in its pass.
struct BlockPlace {
    uint32_t pass, split, tile;  // tile: of the pass's, from 0
    uint32_t row_tile, kv_head, first_member;
};

__device__ __forceinline__ BlockPlace place_block(const AttentionParams& p, uint32_t block) {
    BlockPlace at;
    const uint32_t first = p.pass[0].tiles * p.pass[0].splits;
    at.pass = p.pass_count > 1 && block >= first ? 1u : 0u;
    const AttentionPass& pass = p.pass[at.pass];
    block -= at.pass ? first : 0u;
    at.split = pass.by_tiles.quotient(block, at.tile);
    const uint32_t tile = pass.by_row_tiles.quotient(pass.first_tile + at.tile, at.row_tile);
    at.first_member = p.by_kv_heads.quotient(tile, at.kv_head) * pass.members;
    return at;
}

// Whether the block's rows are whole, and if not, where in the scratch row `row` of its tile (which is row `global_row` of the
// output) goes.
__device__ __forceinline__ bool writes_output(const AttentionParams& p, const BlockPlace& at) { return !p.by_row && p.pass[at.pass].splits == 1; }

__device__ __forceinline__ uint64_t scratch_row(const AttentionParams& p, const BlockPlace& at, uint32_t tile_rows, uint32_t row, uint64_t global_row) {
    return p.by_row ? (p.pass[at.pass].first_slot + at.split) * p.slot_rows + global_row
                    : at.split * p.slot_rows + static_cast<uint64_t>(at.tile) * tile_rows + row;
}

// Where query row r of a pass's group lies.
struct QueryRow {
    uint32_t batch, token, head;
};

__device__ __forceinline__ QueryRow locate_row(const AttentionParams& p, uint32_t first_member, uint32_t kv_head, uint32_t r) {
    uint32_t head, token;
    const uint32_t member = p.by_q_tokens.quotient(p.by_repeat.quotient(r, head), token);
    return {first_member + member, token, kv_head * p.repeat + head};
}

__device__ __forceinline__ uint32_t length_of(const KvView& view, uint32_t slot) {
    if (view.lengths == nullptr) return view.capacity;
    const int32_t length = __ldg(view.lengths + slot);
    return length < 0 ? 0u : min(static_cast<uint32_t>(length), view.capacity);
}

// How many of `length` own keys query `token` sees under the causal mask: the queries are the last q_tokens of the
// sequence. The prefix is seen by all.
__device__ __forceinline__ uint32_t causal_limit(uint32_t length, uint32_t q_tokens, uint32_t token) {
    const int64_t last = static_cast<int64_t>(length) - q_tokens + token + 1;
    return last <= 0 ? 0u : static_cast<uint32_t>(last);
}

// Four bytes of a cache -> two words of FP16 pairs (bytes 0, 1 and bytes 2, 3) without their scale, exact. INT8: the byte
// with its sign bit flipped is q + 128, and 0x6400 | u is the half 1024 + u; E5M2 is the upper byte of a half.
template <int kFormat>
__device__ __forceinline__ uint2 widen4(uint32_t bytes) {
    uint2 r;
    if constexpr (kFormat == KV_INT8) {
        bytes ^= 0x80808080u;
        const __half2 offset = __float2half2_rn(1152.0f);
        const uint32_t lo = __byte_perm(bytes, 0x64646464u, 0x4140), hi = __byte_perm(bytes, 0x64646464u, 0x4342);
        const __half2 a = __hsub2(as_half2(lo), offset), b = __hsub2(as_half2(hi), offset);
        r.x = *reinterpret_cast<const uint32_t*>(&a);
        r.y = *reinterpret_cast<const uint32_t*>(&b);
    } else if constexpr (kFormat == KV_E5M2) {
        r.x = __byte_perm(bytes, 0u, 0x1404);
        r.y = __byte_perm(bytes, 0u, 0x3424);
    } else {
        asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
            : "=r"(r.x), "=r"(r.y) : "r"(bytes));
    }
    return r;
}

// The bits of four bytes of a cache that are not all clear where one of them is not zero.
template <int kFormat>
__device__ __forceinline__ constexpr uint32_t magnitude_bits() { return kFormat == KV_INT8 ? 0xFFFFFFFFu : 0x7F7F7F7Fu; }

// log2 of a value scale, rounded down, as far as it places weights: from 2^-66 on, which also stands for a vector of zeros (what lies
// further down is nothing in a half, whatever the element).
__device__ __forceinline__ float place_bits(float scale) {
    const int exponent = static_cast<int>(__float_as_uint(scale) >> 23 & 0xFFu) - 127;
    return static_cast<float>(max(exponent, -66));
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace sdxlq
