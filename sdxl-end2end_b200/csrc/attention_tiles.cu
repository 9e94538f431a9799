// Attention of many query rows per key head (image tokens, long questions): tiles of 128 rows on the tensor memory. See
// attention.cuh for rows, passes and blocks, attention_rows.cu for few rows.
//
// A CTA takes 128 rows over its share of the keys, in tiles of 64 keys:
//   MMA warp       S = Q K^T (both operands in shared memory), O += P V (P in tensor memory, V as it lies, MN-major);
//                  FP16 keys and values by TMA into a ring of four slots, as SWIZZLE_128B operands
//   loader warps   (8-bit caches) the same through registers, widened to exact halves without their scales
//   softmax warps  a thread per row: S from tensor memory, the weights back into it as halves, in the place of their scores
// Everything that one tile needs of the one before it is a round trip between the warps (softmax, product, scores: 2.2
// thousand clocks, of which the SM's exponentials take 512), so what counts is how many tiles an SM has in flight. Heads of
// 64 take 128 columns of tensor memory and 48 KB, so four CTAs share an SM; heads of up to 128 take 256 columns, two CTAs,
// each with the scores of two tiles. The self-attention of 2 x 4096 tokens, 10 heads of 64,
// takes 145 us (593 TFLOP/s); tiles of 128 keys with two CTAs per SM took 1.6 times as long. Taking every fourth exponential as a
// polynomial on the FMA pipe gave nothing: the pipe of the exponentials is busy half of the time.
//
// With M the row's running reference, a weight is 2^(s_j log2 e - M); M is the running maximum minus 6, and only moves when a
// tile's maximum passes it by more than 2^7: then O, in tensor memory, and the sum are multiplied by 2^(M_old - M). Weights
// of an 8-bit cache are multiplied by their value's scale, and the maximum is that of s_j log2 e + log2(value scale) over the keys
// that the row sees, so that the products are what the halves resolve; O / l is the same for any M.
//
// What bounds it: those round trips; for keys of one or two tiles setting up and storing (5 of 7 us of a CTA's life over 77
// keys: 80 us for 16 x 4096 queries of 10 heads, 2.1 TB/s); for 8-bit caches and heads of 128 the loaders' conversions
// (4 x 333 causal queries over 2333 keys, 16 heads of 80 on 8 in INT8: 86 us). Of these 86 us the search for vectors of zeros takes 4, the
// maximum over score and value scale 2; taken as one product with the key's scale and one sum each it took 10.

#include "attention.cuh"
#include "internal.cuh"
#include "ptx.cuh"

#include <type_traits>
#include <utility>

namespace sdxlq {

namespace {

constexpr uint32_t kTileRows = 128;
constexpr uint32_t kSlots = 4;                   // K0 V0 K1 V1
constexpr uint32_t kScaleRing = 4;               // key tiles whose scales are held
constexpr uint32_t kSoftmaxWarps = 4;
constexpr float kWeightBits = 6.0f, kSlackBits = 7.0f;

// Tensor-memory columns of a CTA: S and, in its place, P (the weights of 32 keys in the first 16 columns of their
// scores), for heads of 128 in two buffers (scores of the next tile under the softmax of this one), then O. Shared memory: Q
// and the ring of slots.
template <int kDim>
struct Shape {
    static constexpr uint32_t kBuffers = kDim == 64 ? 1 : 2;
    static constexpr uint32_t kColumns = kDim == 64 ? 128 : 256;
    static constexpr uint32_t kColumnO = kDim;
    static constexpr uint32_t kTileBytes = kTileKeys * kDim * 2;
    static constexpr uint32_t kQueryBytes = kTileRows * kDim * 2;
};

struct TileControl {
    uint64_t query_ready, score_ready[2], weight_ready[2], value_done[2], vote, drained;       // [j % buffers]: a barrier's parity tells
                                                                                             // one phase from the next only
    uint64_t full[kSlots], empty[kSlots], scales_full[kScaleRing];
    uint32_t tmem_base;
    uint32_t abort;
    uint32_t skip[4];                            // [j % 4] == j + 1: the softmax warps add the values of tile j themselves
};

struct TileParams {
    AttentionParams a;
    AttentionMaps maps;
    uint32_t* error_word;
    long long wait_limit_cycles;
};

// Byte of 16-byte chunk `chunk` of row `row` in a tile of `rows` rows of 128-byte swizzle spans.
__device__ __forceinline__ uint32_t swizzled(uint32_t row, uint32_t chunk, uint32_t rows) {
    return (chunk >> 3) * rows * 128u + row * 128u + (((chunk & 7u) ^ (row & 7u)) << 4);
}

__device__ __forceinline__ float log2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest of three (max.f32 takes three operands on sm_100); NaN never wins.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}

__device__ __forceinline__ bool half_not_finite(uint32_t pair) {
    return (pair & 0x7C00u) == 0x7C00u || (pair & 0x7C000000u) == 0x7C000000u;
}

// The item's place and the tiles of keys that it walks over.
template <int kDim>
struct Item {
    BlockPlace here;
    uint32_t kv_head, first_member, first_row, rows;
    uint32_t prefix_slot, prefix_length, own_length, own_seen;       // own_seen: keys that any row of the tile sees
    uint32_t least_limit;                                            // own keys that all its rows see
    uint32_t prefix_tiles, odd_prefix_tile, odd_own_tiles;           // the odd tile of the prefix; the first odd one of the rest
    uint32_t tile_begin, tile_end;

    __device__ __forceinline__ explicit Item(const AttentionParams& p) {
        here = place_block(p, blockIdx.x);
        const AttentionPass& pass = p.pass[here.pass];
        kv_head = here.kv_head;
        first_member = here.first_member;
        first_row = here.row_tile * kTileRows;
        rows = min(kTileRows, pass.rows - first_row);
        prefix_slot = pass.with_prefix ? p.by_rows_per_prefix.quotient(first_member) : 0u;
        prefix_length = pass.with_prefix ? length_of(p.prefix, prefix_slot) : 0u;
        own_length = own_seen = least_limit = pass.with_own ? length_of(p.own, first_member) : 0u;
        if (p.causal && pass.with_own) {
            own_seen = causal_limit(own_length, p.q_tokens, p.by_repeat.quotient(first_row + rows - 1));
            least_limit = causal_limit(own_length, p.q_tokens, p.by_repeat.quotient(first_row));
        }
        prefix_tiles = (prefix_length + kTileKeys - 1) / kTileKeys;
        odd_prefix_tile = prefix_length % kTileKeys != 0 ? prefix_tiles - 1 : ~0u;
        odd_own_tiles = prefix_tiles + least_limit / kTileKeys;
        tile_begin = 0;
        tile_end = prefix_tiles + (own_seen + kTileKeys - 1) / kTileKeys;
        if (pass.splits != 1) {
            const uint64_t tiles = tile_end;
            tile_begin = static_cast<uint32_t>(tiles * here.split / pass.splits);
            tile_end = static_cast<uint32_t>(tiles * (here.split + 1) / pass.splits);
        }
    }

    // Every row sees every key of the tile.
    __device__ __forceinline__ bool ordinary(uint32_t index) const { return index != odd_prefix_tile && index < odd_own_tiles; }

    struct Tile {
        bool in_prefix;
        uint32_t first, end;         // first key of the tile, end of the part's keys
        uint32_t columns;            // keys of the tile, rounded up to the MMA's 16
    };
    __device__ __forceinline__ Tile tile(uint32_t index) const {
        Tile t;
        t.in_prefix = index < prefix_tiles;
        t.first = (t.in_prefix ? index : index - prefix_tiles) * kTileKeys;
        t.end = t.in_prefix ? prefix_length : own_seen;
        t.columns = min(kTileKeys, (t.end - t.first + 15u) & ~15u);
        return t;
    }
};

template <int kDim, int kFormat, int kLoaderWarps, int kBlocks>
__global__ void __launch_bounds__(32 * (kSoftmaxWarps + 1 + kLoaderWarps), kBlocks) attention_tiles_kernel(const __grid_constant__ TileParams params) {
    using S = Shape<kDim>;
    constexpr uint32_t kBuffers = S::kBuffers;
    constexpr bool kScaled = kFormat != KV_F16;
    const AttentionParams& p = params.a;
    extern __shared__ __align__(1024) uint8_t dynamic_smem[];
    __shared__ TileControl control;
    // key scales * softmax scale, value scales (0: a vector of zeros), and log2 of the latter as place_bits has it
    __shared__ __align__(16) float scales[kScaled ? kScaleRing : 1][3][kScaled ? kTileKeys : 1];
    const uint32_t query_base = ptx::smem_u32(dynamic_smem), slots_base = query_base + S::kQueryBytes;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    volatile uint32_t* const abort_word = &control.abort;
    const long long limit = params.wait_limit_cycles;

    wait_for_prior_kernels_then_release_next();
    const Item<kDim> item(p);
    const uint32_t tiles = item.tile_end - item.tile_begin;
    const uint32_t full = ptx::smem_u32(&control.full[0]), empty = ptx::smem_u32(&control.empty[0]);
    const auto give_up = [&](uint32_t code) {
        *abort_word = 1;
        atomicCAS(params.error_word, 0u, code);
    };

    // FP16 keys (0) and values (1), a tile at a time, by the MMA warp
    uint32_t loaded[2] = {0, 0};
    const auto load_tile = [&](uint32_t which) {
        if (kScaled || loaded[which] == tiles) return;
        const uint32_t index = loaded[which]++, slot = (2 * index + which) % kSlots, bar = full + slot * 8u;
        const typename Item<kDim>::Tile t = item.tile(item.tile_begin + index);
        if (ptx::elect_one()) {
            const uint32_t part = t.in_prefix ? 0u : 1u, sequence = t.in_prefix ? item.prefix_slot : item.first_member;
            ptx::mbar_expect_tx(bar, S::kTileBytes);
#pragma unroll
            for (uint32_t d = 0; d < kDim; d += 64) {
                ptx::tma_load_4d(slots_base + slot * S::kTileBytes + d * (kTileKeys * 2), &params.maps.map[part][which], bar, static_cast<int32_t>(d),
                                 static_cast<int32_t>(item.kv_head), static_cast<int32_t>(t.first), static_cast<int32_t>(sequence));
            }
        }
        __syncwarp();
    };

    // Q and the output move by whole lines: a lane takes 16 bytes of the warp's rows in turn, eight at a time. The first eight
    // are on their way while the barriers and the tensor memory are set up.
    constexpr uint32_t kChunksOfRow = kDim / 8, kRowsAtOnce = 32 / kChunksOfRow, kBatch = 8;
    const uint32_t row = threadIdx.x;                                    // of the tile, and lane of tensor memory (softmax)
    const uint32_t chunk_of_row = lane % kChunksOfRow, first_of_warp = warp * 32u + lane / kChunksOfRow;
    const bool in_head = chunk_of_row * 8u < p.dim;
    QueryRow at{};
    int64_t query_offset = 0;
    uint4 query[kBatch];
    const auto load_queries = [&](uint32_t first) {
#pragma unroll
        for (uint32_t i = 0; i < kBatch; ++i) {
            const uint32_t r = first_of_warp + first + i * kRowsAtOnce;
            const int64_t from = __shfl_sync(0xffffffffu, query_offset, r & 31u);
            query[i] = r < item.rows && in_head ? __ldg(reinterpret_cast<const uint4*>(p.q + from + chunk_of_row * 8u)) : make_uint4(0u, 0u, 0u, 0u);
        }
    };
    if (warp < kSoftmaxWarps) {
        at = locate_row(p, item.first_member, item.kv_head, item.first_row + min(row, item.rows - 1));
        query_offset = at.batch * p.q_batch + at.token * p.q_token + at.head * p.q_head;
        load_queries(0);
        if (threadIdx.x == 0) {
            ptx::mbar_init(ptx::smem_u32(&control.query_ready), kSoftmaxWarps);
            for (uint32_t b = 0; b < kBuffers; ++b) {
                ptx::mbar_init(ptx::smem_u32(&control.score_ready[b]), 1);
                ptx::mbar_init(ptx::smem_u32(&control.weight_ready[b]), kSoftmaxWarps);
                ptx::mbar_init(ptx::smem_u32(&control.value_done[b]), 1);
            }
            ptx::mbar_init(ptx::smem_u32(&control.vote), kSoftmaxWarps);
            ptx::mbar_init(ptx::smem_u32(&control.drained), 1);
            for (uint32_t s = 0; s < kScaleRing; ++s) ptx::mbar_init(ptx::smem_u32(&control.scales_full[s]), kScaled ? kLoaderWarps : 1);
            for (uint32_t s = 0; s < kSlots; ++s) {
                ptx::mbar_init(full + s * 8u, kScaled ? kLoaderWarps : 1);
                ptx::mbar_init(empty + s * 8u, 1);
            }
            control.abort = 0;
            for (uint32_t i = 0; i < 4; ++i) control.skip[i] = 0;
            ptx::fence_mbar_init();
        }
    } else if (warp == kSoftmaxWarps) {
        ptx::tmem_alloc(ptx::smem_u32(&control.tmem_base), S::kColumns);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before();
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&control.tmem_base);

    if (warp > kSoftmaxWarps) {
        // ---------------------------------------- loaders ----------------------------------------
        const uint32_t thread = threadIdx.x - 32u * (kSoftmaxWarps + 1);
        constexpr uint32_t kThreads = 32u * kLoaderWarps;
        const auto slot_free = [&](uint32_t unit) {
            return ptx::warp_wait_bounded(empty + (unit % kSlots) * 8u, ((unit / kSlots) & 1u) ^ 1u, abort_word, limit);
        };
        const auto announce = [&](uint32_t unit) {
            ptx::fence_proxy_async();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(full + (unit % kSlots) * 8u);
        };
        if constexpr (kScaled) {
            constexpr uint32_t kChunks = kDim / 16;                      // 16-byte loads of a key
            constexpr uint32_t kStep = kThreads / kChunks;
            constexpr uint32_t kRounds = (kTileKeys + kStep - 1) / kStep;
            constexpr uint32_t kAhead = 2;
            static_assert(kThreads % kChunks == 0);
            const uint32_t chunk = thread % kChunks, first_key = thread / kChunks;
            const bool in_head = chunk * 16u < p.dim;
            // kAhead tiles of K or V are on their way to the registers at a time
            uint4 ahead[kAhead][kRounds];
            // a lane has the scales of one of the keys that its warp loads in a tile
            constexpr uint32_t kKeysOfRound = 32 / kChunks;
            static_assert(kAhead == 2 && kRounds * kKeysOfRound <= 32);
            const uint32_t scale_round = lane / kKeysOfRound, scale_key = scale_round * kStep + thread / 32u * kKeysOfRound + lane % kKeysOfRound;
            const bool has_scale = scale_round < kRounds && scale_key < kTileKeys;
            float ahead_scale[kAhead] = {};
            // where the thread's first 16 bytes of the next tile to fetch are, in K and V, and its scales; tiles come in order
            const uint8_t* from[2] = {};
            const float* scale_from[2] = {};
            int64_t step = 0, to_next = 0;                               // bytes between rounds, and from tile to tile
            typename Item<kDim>::Tile t{};
            const auto seek = [&](uint32_t index) {
                const bool was_in_prefix = t.in_prefix;
                t = item.tile(item.tile_begin + index);
                if (index != 0 && was_in_prefix == t.in_prefix) {
                    from[0] += to_next; from[1] += to_next;
                    scale_from[0] += kTileKeys; scale_from[1] += kTileKeys;
                    return;
                }
                const KvView& view = t.in_prefix ? p.prefix : p.own;
                const int64_t sequence = t.in_prefix ? item.prefix_slot : item.first_member;
                const int64_t at = sequence * view.slot_stride + item.kv_head * view.head_stride + static_cast<int64_t>(t.first + first_key) * view.token_stride + chunk * 16u;
                const int64_t scales_at = (sequence * p.kv_heads + item.kv_head) * view.capacity + t.first;
                from[0] = view.k + at;
                from[1] = view.v + at;
                scale_from[0] = view.k_scales + scales_at;
                scale_from[1] = view.v_scales + scales_at;
                step = kStep * view.token_stride;
                to_next = kTileKeys * view.token_stride;
            };
            const auto fetch = [&](uint32_t unit, auto buffer) {
                constexpr uint32_t kBuffer = decltype(buffer)::value, kWhich = kBuffer % 2;
                if constexpr (kWhich == 0) seek(unit / 2);
                const uint8_t* at = from[kWhich];
                const uint32_t left = min(t.end - t.first, kTileKeys);
#pragma unroll
                for (uint32_t i = 0; i < kRounds; ++i, at += step) {
                    const bool inside = in_head && first_key + i * kStep < left;
                    ahead[kBuffer][i] = inside ? __ldg(reinterpret_cast<const uint4*>(at)) : make_uint4(0u, 0u, 0u, 0u);
                }
                const float scale = has_scale && scale_key < left ? __ldg(scale_from[kWhich] + scale_key) : 0.0f;
                ahead_scale[kWhich] = kWhich == 0 ? scale * fabsf(p.scale_log2) : scale;
            };
            const auto put = [&](uint32_t unit, auto buffer) {
                constexpr uint32_t kBuffer = decltype(buffer)::value;
                if (!slot_free(unit)) return false;
                const uint32_t to = slots_base + (unit % kSlots) * S::kTileBytes;
#pragma unroll
                for (uint32_t i = 0; i < kRounds; ++i) {
                    const uint32_t key = first_key + i * kStep;
                    if (key >= kTileKeys) break;
                    const uint4 x = ahead[kBuffer][i];
                    const uint2 a = widen4<kFormat>(x.x), b = widen4<kFormat>(x.y), c = widen4<kFormat>(x.z), d = widen4<kFormat>(x.w);
                    ptx::st_shared16(to + swizzled(key, 2u * chunk, kTileKeys), make_uint4(a.x, a.y, b.x, b.y));
                    ptx::st_shared16(to + swizzled(key, 2u * chunk + 1u, kTileKeys), make_uint4(c.x, c.y, d.x, d.y));
                }
                // The ring of scales is as long as its writer can be ahead of its readers: this tile's slot was freed by the MMA
                // of the tile two before it, and that had waited for the weights of the tile kBuffers before it.
                static_assert(kScaleRing >= kSlots / 2 + kBuffers);
                auto& ring = scales[unit / 2 % kScaleRing];
                if constexpr (kBuffer % 2 == 0) {
                    if (has_scale) ring[0][scale_key] = ahead_scale[0];
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&control.scales_full[unit / 2 % kScaleRing]));
                } else {
                    // A vector of zeros adds nothing whatever its scale is (1, where the cache was written from zeros), and must
                    // not be what the other weights are placed by: its scale becomes 0.
                    uint32_t lives = 0;
#pragma unroll
                    for (uint32_t i = 0; i < kRounds; ++i) {
                        const uint4 x = ahead[kBuffer][i];
                        const uint32_t some = __ballot_sync(0xffffffffu, ((x.x | x.y | x.z | x.w) & magnitude_bits<kFormat>()) != 0);
                        if (scale_round == i) lives = some;
                    }
                    lives = lives >> (lane % kKeysOfRound * kChunks) & ((1u << kChunks) - 1u);
                    if (has_scale) {
                        const float scale = lives != 0 ? ahead_scale[1] : 0.0f;
                        ring[1][scale_key] = scale;
                        ring[2][scale_key] = place_bits(scale);
                    }
                }
                if (unit + kAhead < 2 * tiles) fetch(unit + kAhead, buffer);
                announce(unit);
                return true;
            };
            // buffer by buffer, each known at compile time
            const auto each_buffer = [&](auto action) {
                [&]<uint32_t... kBuffer>(std::integer_sequence<uint32_t, kBuffer...>) {
                    return (action(std::integral_constant<uint32_t, kBuffer>{}) && ...);
                }(std::make_integer_sequence<uint32_t, kAhead>{});
            };
            each_buffer([&](auto buffer) {
                if (buffer.value < 2 * tiles) fetch(buffer.value, buffer);
                return true;
            });
            bool ok = true;
            for (uint32_t first = 0; ok && first < 2 * tiles; first += kAhead) {
                each_buffer([&](auto buffer) {
                    if (first + buffer.value < 2 * tiles) ok = put(first + buffer.value, buffer);
                    return ok;
                });
            }
            if (!ok) give_up(DEV_TIMEOUT_PRODUCER);
        }
    } else if (warp == kSoftmaxWarps) {
        // ------------------------- MMA issuer, and the loads of FP16 keys and values -------------------------
        const auto wait = [&](const uint64_t& bar, uint32_t parity) {
            return ptx::warp_wait_bounded(ptx::smem_u32(&bar), parity, abort_word, limit);
        };
        const auto wait_full = [&](uint32_t unit) {
            return ptx::warp_wait_bounded(full + (unit % kSlots) * 8u, (unit / kSlots) & 1u, abort_word, limit);
        };
        // V is the B operand with its head dimension together (MN-major: bit 16); 64 of it to an MMA
        constexpr uint32_t kValueIdesc = ptx::umma_instr_desc(1, 0, 0, kTileRows, 64) | (1u << 16);
        const uint32_t query_lo = ptx::umma_desc_lo(query_base), slots_lo = ptx::umma_desc_lo(slots_base);
        const auto multiply_scores = [&](uint32_t j) {
            const uint32_t slot = 2 * j % kSlots, columns = item.tile(item.tile_begin + j).columns;
            const uint32_t idesc = ptx::umma_instr_desc(1, 0, 0, kTileRows, columns);
            if (ptx::elect_one()) {
                const uint32_t b = slots_lo + slot * (S::kTileBytes / 16);
#pragma unroll
                for (uint32_t part = 0; part < kDim / 64; ++part) {
                    ptx::umma_stage_f16(tmem + j % kBuffers * kTileKeys, query_lo + part * (kTileRows * 128 / 16), b + part * (kTileKeys * 128 / 16),
                                        ptx::kUmmaDescHiSw128, idesc, part);
                }
                if (kScaled) ptx::umma_commit(empty + slot * 8u);
                ptx::umma_commit(ptx::smem_u32(&control.score_ready[j % kBuffers]));
            }
            __syncwarp();
        };
        for (uint32_t i = 0; i < 4; ++i) load_tile(i % 2);
        bool ok = tiles == 0 || wait(control.query_ready, 0);
        for (uint32_t j = 0; ok && j < min(tiles, kBuffers); ++j) {
            ok = wait_full(2 * j);
            ptx::tc_fence_after();
            if (ok) multiply_scores(j);
        }
        for (uint32_t j = 0; ok && j < tiles; ++j) {
            const uint32_t unit = 2 * j + 1, slot = unit % kSlots, columns = item.tile(item.tile_begin + j).columns;
            const uint32_t buffer = j % kBuffers, phase = (j / kBuffers) & 1u, next = j + kBuffers;
            if (!kScaled) {
                ok = wait(control.score_ready[buffer], phase);           // the keys of tile j have been read: the next but one take their slot
                if (!ok) break;
                load_tile(0);
            }
            ok = wait_full(unit) && (next >= tiles || wait_full(2 * next)) && wait(control.weight_ready[buffer], phase);
            if (!ok) break;
            ptx::tc_fence_after();
            const bool skip = kFormat != KV_INT8 && p.causal && *reinterpret_cast<volatile uint32_t*>(&control.skip[j % 4]) == j + 1;
            if (ptx::elect_one()) {
                const uint32_t b = slots_lo + slot * (S::kTileBytes / 16), a = tmem + buffer * kTileKeys;
#pragma unroll
                for (uint32_t part = 0; part < kDim / 64; ++part) {
                    const uint32_t d = tmem + S::kColumnO + part * 64, b_part = b + part * (kTileKeys * 128 / 16);
                    if (skip) break;
                    if (columns == kTileKeys) {
                        ptx::umma_f16_ts_x4(d, a, b_part, ptx::kUmmaDescHiSw128, kValueIdesc, j);
                    } else {
                        for (uint32_t step = 0; step < columns / 16; ++step) {
                            ptx::umma_f16_ts(d, a + step / 2 * 32 + step % 2 * 8, b_part + step * (16 * 128 / 16), ptx::kUmmaDescHiSw128, kValueIdesc,
                                             j | step);
                        }
                    }
                }
                if (kScaled) ptx::umma_commit(empty + slot * 8u);
                ptx::umma_commit(ptx::smem_u32(&control.value_done[buffer]));
            }
            __syncwarp();
            if (next < tiles || loaded[1] < tiles) {
                ok = wait(control.value_done[buffer], phase);            // P has been read: S may take its place, and values the slot
                ptx::tc_fence_after();
                if (ok && next < tiles) multiply_scores(next);
                if (ok) load_tile(1);
            }
        }
        if (!ok) {
            give_up(DEV_TIMEOUT_MMA);
            if (ptx::elect_one()) ptx::umma_commit(ptx::smem_u32(&control.drained));         // what was issued ends before its memory goes
            __syncwarp();
            uint32_t never = 0;
            ptx::mbar_wait_bounded(ptx::smem_u32(&control.drained), 0, &never, limit);
            for (uint32_t which = 0; which < 2; ++which) {               // and so do the copies
                for (uint32_t index = loaded[which] > 2 ? loaded[which] - 2 : 0; index < loaded[which]; ++index) {
                    const uint32_t unit = 2 * index + which;
                    ptx::mbar_wait_bounded(full + (unit % kSlots) * 8u, (unit / kSlots) & 1u, &never, limit);
                }
            }
        }
    } else {
        // ---------------------------------------- softmax ----------------------------------------
        const uint32_t my_tmem = tmem + ((warp * 32u) << 16);
        const uint32_t column_o = my_tmem + S::kColumnO;
        const bool warp_active = warp * 32u < item.rows;
        const auto wait = [&](const uint64_t& bar, uint32_t parity) {
            return ptx::warp_wait_bounded(ptx::smem_u32(&bar), parity, abort_word, limit);
        };
        const auto arrive = [&](uint64_t& bar) {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(ptx::smem_u32(&bar));
        };
        {
            // a negative softmax scale turns the queries' signs, so that scores are multiplied by its magnitude
            const uint32_t flip = p.scale_log2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
            for (uint32_t first = 0; first < 32; first += kBatch * kRowsAtOnce) {
                if (first != 0) load_queries(first);
#pragma unroll
                for (uint32_t i = 0; i < kBatch; ++i) {
                    uint4 x = query[i];
                    x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
                    ptx::st_shared16(query_base + swizzled(first_of_warp + first + i * kRowsAtOnce, chunk_of_row, kTileRows), x);
                }
            }
            ptx::fence_proxy_async();
            arrive(control.query_ready);
        }
        const float scale = fabsf(p.scale_log2);
        const uint32_t own_limit = p.causal ? causal_limit(item.own_length, p.q_tokens, at.token) : item.own_length;
        const float kNone = __int_as_float(0xff800000);
        float reference = kNone, fine = 0.0f, sum = 0.0f;
        bool huge = false;                                               // some row's reference is coarser than the weights' room
        uint32_t votes = 0;
        bool ok = true;
        for (uint32_t j = 0; j < tiles; ++j) {
            const bool masked = !item.ordinary(item.tile_begin + j);
            uint32_t columns = kTileKeys, visible = kTileKeys, values = kTileKeys;       // of the tile; that this row sees; that exist
            bool ragged = false;                                         // rows differ in what they see of the tile
            if (masked) {
                const typename Item<kDim>::Tile t = item.tile(item.tile_begin + j);
                const uint32_t seen = t.in_prefix ? item.prefix_length : own_limit;
                columns = t.columns;
                values = min(t.end - t.first, kTileKeys);
                visible = seen > t.first ? min(seen - t.first, kTileKeys) : 0u;
                ragged = p.causal && !t.in_prefix;
            }
            const float* const key_scales = scales[j % kScaleRing][0];
            const float* const value_scales = scales[j % kScaleRing][kScaled ? 1 : 0];
            const float* const value_bits = scales[j % kScaleRing][kScaled ? 2 : 0];
            if (kScaled) {                                               // the values' scales come with the values
                ok = wait(control.scales_full[j % kScaleRing], (j / kScaleRing) & 1u) &&
                     wait(control.full[(2 * j + 1) % kSlots], ((2 * j + 1) / kSlots) & 1u);
            }
            ok = ok && wait(control.score_ready[j % kBuffers], (j / kBuffers) & 1u);
            const uint32_t column_s = my_tmem + j % kBuffers * kTileKeys;
            if (!ok) break;
            ptx::tc_fence_after();

            // 32 columns of S; an 8-bit cache's without their key's scale, which the fused multiply-adds below bring in
            const auto load = [&](uint32_t c, uint32_t (&s)[32]) {
                ptx::tmem_ld_32x32b_x32(column_s + c * 32u, s);
                ptx::tmem_ld_wait(s);
            };
            // the largest of 32 columns: of the scores in FP16 without their scale, which is the same for all; of an 8-bit cache's
            // scores plus the logarithm of their value's scale
            const auto largest_of = [&](auto careful_case, uint32_t c, const uint32_t (&s)[32], float largest) {
                constexpr bool careful = decltype(careful_case)::value;
                float other = largest;
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    float x[4] = {__uint_as_float(s[i]), __uint_as_float(s[i + 1]), __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])};
                    if constexpr (kScaled) {
                        const float4 k = *reinterpret_cast<const float4*>(key_scales + c * 32u + i), bits = *reinterpret_cast<const float4*>(value_bits + c * 32u + i);
                        const float2 lo = __ffma2_rn(make_float2(x[0], x[1]), make_float2(k.x, k.y), make_float2(bits.x, bits.y));
                        const float2 hi = __ffma2_rn(make_float2(x[2], x[3]), make_float2(k.z, k.w), make_float2(bits.z, bits.w));
                        x[0] = lo.x; x[1] = lo.y; x[2] = hi.x; x[3] = hi.y;
                    }
                    if (careful) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] = c * 32u + i + e < visible ? x[e] : kNone;
                    }
                    largest = max3(largest, x[0], x[1]);
                    other = max3(other, x[2], x[3]);
                }
                return max3(largest, other, other);
            };
            // the weights of 32 columns: into P, and into the row's sum
            const auto weigh = [&](auto careful_case, uint32_t c, const uint32_t (&s)[32], float shift, float2 (&part)[2]) {
                constexpr bool careful = decltype(careful_case)::value;
                uint32_t w[16];
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    // Scores in units of log2, less the reference. The fused multiply-add rounds the difference alone, so that
                    // it is as exact for large scores as for small ones.
                    float2 lo = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), hi = make_float2(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
                    const float2 back = make_float2(-shift, -shift);
                    float4 k = make_float4(scale, scale, scale, scale);
                    if constexpr (kScaled) k = *reinterpret_cast<const float4*>(key_scales + c * 32u + i);
                    lo = __ffma2_rn(lo, make_float2(k.x, k.y), back);
                    hi = __ffma2_rn(hi, make_float2(k.z, k.w), back);
                    float x[4] = {lo.x, lo.y, hi.x, hi.y};
                    if (careful) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[e] -= fine;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (careful) x[e] = c * 32u + i + e < visible ? x[e] : kNone;
                        x[e] = exp2_approx(x[e]);
                    }
                    part[0] = __fadd2_rn(part[0], make_float2(x[0], x[1]));
                    part[1] = __fadd2_rn(part[1], make_float2(x[2], x[3]));
                    if constexpr (kScaled) {
                        const float4 v = *reinterpret_cast<const float4*>(value_scales + c * 32u + i);
                        const float2 a = __fmul2_rn(make_float2(x[0], x[1]), make_float2(v.x, v.y)), b = __fmul2_rn(make_float2(x[2], x[3]), make_float2(v.z, v.w));
                        x[0] = a.x; x[1] = a.y; x[2] = b.x; x[3] = b.y;
                        if (careful) {                                   // a hidden key's scale may be anything
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[e] = c * 32u + i + e < visible ? x[e] : 0.0f;
                        }
                    }
                    w[i / 2] = pack_half2(x[0], x[1]);
                    w[i / 2 + 1] = pack_half2(x[2], x[3]);
                }
                ptx::tmem_st_32x32b_x16(column_s + c * 32u, w);
            };
            // O is whole when the products of the tile before are done; with one buffer the scores' MMA has come behind them.
            const auto values_done = [&] {
                if (kBuffers == 1 || j == 0) return true;
                const bool done = wait(control.value_done[(j - 1) % kBuffers], ((j - 1) / kBuffers) & 1u);
                ptx::tc_fence_after();
                return done;
            };
            if (warp_active) {
                const bool both = columns > 32u;
                // Columns 32 to 63 stay in registers until they are weighed; the first 32 too, where there is room for them.
                constexpr bool kHold = kDim > 64;
                uint32_t s[kHold ? 2 : 1][32];
                uint32_t (&s0)[32] = s[0], (&s1)[32] = s[kHold ? 1 : 0];
                float largest = kNone;
                const auto find_largest = [&](auto careful) {
                    load(0, s0);
                    largest = largest_of(careful, 0, s0, largest);
                    if (both) {
                        load(1, s1);
                        largest = largest_of(careful, 1, s1, largest);
                    }
                };
                if (masked) find_largest(std::true_type{});
                else find_largest(std::false_type{});
                // the reference moves where the tile's largest weight would be 2^7 past its place, and in the row's first tile
                const float unit = kScaled ? 1.0f : scale;
                const bool first = reference == kNone && largest > kNone;
                float base = first ? largest * unit : reference;
                float over = fmaf(largest, unit, -base);
                if constexpr (kScaled) {
                    // The sum of such a score and a logarithm is rounded too coarsely to place a weight by. Differences of scores
                    // are exact: again, with the largest score for the reference of a first tile.
                    if (__any_sync(0xffffffffu, largest > kNone && fabsf(largest) > 1048576.0f)) {
                        float top = kNone;
                        over = kNone;
                        for (uint32_t pass = 0; pass < 2; ++pass) {
                            for (uint32_t c = 0; c < (both ? 2u : 1u); ++c) {
                                load(c, s0);
#pragma unroll
                                for (uint32_t i = 0; i < 32; ++i) {
                                    const float x = fmaf(__uint_as_float(s0[i]), key_scales[c * 32u + i], pass == 0 ? 0.0f : -base);
                                    if (c * 32u + i >= visible) continue;
                                    if (pass == 0) top = fmaxf(top, x);
                                    else over = fmaxf(over, x + value_bits[c * 32u + i]);
                                }
                            }
                            base = first ? top : reference;
                        }
                        if (largest == kNone) over = kNone;
                        if (kHold) load(0, s0);                          // s1 is as it was; one buffer has its last columns again
                    }
                }
                over -= fine + kWeightBits;
                const bool moves = first || over > kSlackBits;
                if (__any_sync(0xffffffffu, moves)) {
                    float grow = 1.0f;
                    if (moves) {
                        // the last bit of a reference past 2^22 is coarser than the weights' room: what it rounds off is kept too
                        const float step = fine + over, moved = base + step, back = moved - base;
                        const float rest = fabsf(moved) > 4194304.0f ? (base - (moved - back)) + (step - back) : 0.0f;
                        grow = exp2_approx((reference - moved) + (fine - rest));
                        reference = moved;
                        fine = rest;
                        sum *= grow;
                    }
                    huge = __any_sync(0xffffffffu, fabsf(reference) > 4194304.0f && reference != kNone);
                    if (j != 0) {
                        ok = values_done();
                        if (!ok) break;
#pragma unroll
                        for (uint32_t c = 0; c < kDim; c += 16) {
                            uint32_t o[16];
                            ptx::tmem_ld_32x32b_x16(column_o + c, o);
                            ptx::tmem_ld_wait(o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * grow);
                            ptx::tmem_st_32x32b_x16(column_o + c, o);
                        }
                    }
                }
                float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                const float shift = reference == kNone ? 0.0f : reference;       // a row that has seen nothing has no weights at all
                const auto take_weights = [&](auto careful) {
                    if (both) {
                        weigh(careful, 1, s1, shift, part);
                        if (!kHold) load(0, s0);
                    }
                    weigh(careful, 0, s0, shift, part);
                };
                if (masked || huge) take_weights(std::true_type{});
                else take_weights(std::false_type{});
                sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
            }
            ptx::tmem_st_wait();

            // What lies behind the end of a part, within the MMA's last 16 keys, was loaded as it is: zeros take its place, since
            // 0 * v is not 0 for every v. (Loader warps put zeros there themselves.)
            if (!kScaled && values < columns) {
                const uint32_t unit = 2 * j + 1, base = slots_base + (unit % kSlots) * S::kTileBytes;
                ok = wait(control.full[unit % kSlots], (unit / kSlots) & 1u);
                if (!ok) break;
                for (uint32_t i = threadIdx.x; i < (columns - values) * (kDim / 8); i += 32 * kSoftmaxWarps) {
                    ptx::st_shared16(base + swizzled(values + i / (kDim / 8), i % (kDim / 8), kTileKeys), make_uint4(0u, 0u, 0u, 0u));
                }
                ptx::fence_proxy_async();
            }

            // A value that is not finite makes 0 * v a NaN, also in rows that the causal mask hides it from (what lies behind
            // a length is zeros by now). Tiles that such a mask divides are looked through, and one that holds such a value
            // is multiplied here, row by row over the keys that the row sees.
            if (kFormat != KV_INT8 && ragged) {
                const uint32_t unit = 2 * j + 1, base = slots_base + (unit % kSlots) * S::kTileBytes;
                volatile uint32_t* const skip = &control.skip[j % 4];
                ok = values_done() && wait(control.full[unit % kSlots], (unit / kSlots) & 1u);
                if (!ok) break;
                bool found = false;
                // the keys that exist: other warps may still be putting the zeros behind them
                for (uint32_t i = threadIdx.x; i < values * (kDim / 8); i += 32 * kSoftmaxWarps) {
                    const uint4 x = ptx::ld_shared16(base + swizzled(i / (kDim / 8), i % (kDim / 8), kTileKeys));
                    found = found || half_not_finite(x.x) || half_not_finite(x.y) || half_not_finite(x.z) || half_not_finite(x.w);
                }
                if (found) *skip = j + 1;
                arrive(control.vote);
                ok = wait(control.vote, votes & 1u);
                if (!ok) break;
                ++votes;
                if (*skip == j + 1 && warp_active) {
                    for (uint32_t c = 0; c < kDim; c += 8) {
                        uint32_t o[8];
                        ptx::tmem_ld_32x32b_x8(column_o + c, o);
                        ptx::tmem_ld_wait(o);
                        float total[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) total[i] = j == 0 ? 0.0f : __uint_as_float(o[i]);
                        for (uint32_t key = 0; key < values; ++key) {
                            uint32_t pair;
                            ptx::tmem_ld_32x32b_x1(column_s + key / 32 * 32 + key % 32 / 2, pair);
                            ptx::tmem_ld_wait(pair);
                            const float w = key % 2 == 0 ? half_lo(pair) : half_hi(pair);
                            const uint4 x = ptx::ld_shared16(base + swizzled(key, c / 8, kTileKeys));
                            if (key < visible) {
                                total[0] = fmaf(w, half_lo(x.x), total[0]); total[1] = fmaf(w, half_hi(x.x), total[1]);
                                total[2] = fmaf(w, half_lo(x.y), total[2]); total[3] = fmaf(w, half_hi(x.y), total[3]);
                                total[4] = fmaf(w, half_lo(x.z), total[4]); total[5] = fmaf(w, half_hi(x.z), total[5]);
                                total[6] = fmaf(w, half_lo(x.w), total[6]); total[7] = fmaf(w, half_hi(x.w), total[7]);
                            }
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) o[i] = __float_as_uint(total[i]);
                        ptx::tmem_st_32x32b_x8(column_o + c, o);
                    }
                    ptx::tmem_st_wait();
                }
            }
            arrive(control.weight_ready[j % kBuffers]);
        }
        // from here on the room of Q is free: the last product has read it, or (no keys) all warps have written theirs
        if (ok && tiles == 0) ok = wait(control.query_ready, 0);
        if (ok && tiles != 0) ok = wait(control.value_done[(tiles - 1) % kBuffers], ((tiles - 1) / kBuffers) & 1u);
        ptx::tc_fence_after();
        if (!ok) {
            give_up(DEV_TIMEOUT_EPILOGUE);
        } else if (warp_active) {
            const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
            const bool nothing = tiles == 0 || sum == 0.0f;              // O was never written, or holds no weight
            if (writes_output(p, item.here)) {
                // the warp's rows of Q make room for its rows of the output, which leave in whole lines
#pragma unroll
                for (uint32_t c = 0; c < kDim; c += 16) {
                    uint32_t o[16];
                    ptx::tmem_ld_32x32b_x16(column_o + c, o);
                    ptx::tmem_ld_wait(o);
                    float x[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = nothing ? 0.0f : __uint_as_float(o[i]) * inverse;
                    ptx::st_shared16(query_base + swizzled(row, c / 8, kTileRows),
                                     make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7])));
                    ptx::st_shared16(query_base + swizzled(row, c / 8 + 1, kTileRows),
                                     make_uint4(pack_half2(x[8], x[9]), pack_half2(x[10], x[11]), pack_half2(x[12], x[13]), pack_half2(x[14], x[15])));
                }
                __syncwarp();
                const int64_t offset = at.batch * p.y_batch + at.token * p.y_token + at.head * p.y_head;
#pragma unroll 8
                for (uint32_t i = 0; i < 32; i += kRowsAtOnce) {
                    const uint32_t r = first_of_warp + i;
                    const int64_t to = __shfl_sync(0xffffffffu, offset, r & 31u);
                    if (r < item.rows && in_head) *reinterpret_cast<uint4*>(p.y + to + chunk_of_row * 8u) = ptx::ld_shared16(query_base + swizzled(r, chunk_of_row, kTileRows));
                }
            } else {
                // in 32 bits through the warp's share of the slots, which are free by now, and out in whole lines
                const uint64_t place = scratch_row(p, item.here, kTileRows, row, (static_cast<uint64_t>(at.batch) * p.q_tokens + at.token) * p.q_heads + at.head);
                constexpr uint32_t kQuads = kDim / 4, kRowsOut = 32 / kQuads;
                const uint32_t room = slots_base + warp * (32 * kDim * 4);
#pragma unroll
                for (uint32_t c = 0; c < kDim; c += 16) {
                    uint32_t o[16];
                    ptx::tmem_ld_32x32b_x16(column_o + c, o);
                    ptx::tmem_ld_wait(o);
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = nothing ? 0u : __float_as_uint(__uint_as_float(o[i]) * inverse);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        ptx::st_shared16(room + lane * (kDim * 4) + (((c / 4 + i) ^ (lane & 7u)) << 4), make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]));
                    }
                }
                __syncwarp();
                const uint32_t quad = lane % kQuads;
#pragma unroll 8
                for (uint32_t r = lane / kQuads; r < 32; r += kRowsOut) {
                    const uint64_t to = __shfl_sync(0xffffffffu, place, r);
                    const uint4 x = ptx::ld_shared16(room + r * (kDim * 4) + ((quad ^ (r & 7u)) << 4));
                    if (warp * 32u + r < item.rows && quad * 4u < p.dim) *reinterpret_cast<uint4*>(p.part_o + to * p.dim + quad * 4u) = x;
                }
                if (row < item.rows) p.part_lse[place] = make_float2(sum == 0.0f ? kNone : reference > kNone ? reference : 0.0f, fine + log2f(sum));
            }
        }
    }
    ptx::tc_fence_before();
    __syncthreads();
    if (warp == kSoftmaxWarps) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem, S::kColumns);
    }
}

template <int kDim, int kFormat>
cudaError_t launch_tiles(const TileParams& params, cudaStream_t stream, bool early_launch) {
    constexpr int kLoaderWarps = kFormat == KV_F16 ? 0 : kDim == 64 ? 2 : 3;
    constexpr int kBlocks = static_cast<int>(tile_blocks_per_sm(kDim, static_cast<KvFormat>(kFormat)));
    constexpr size_t bytes = Shape<kDim>::kQueryBytes + kSlots * Shape<kDim>::kTileBytes;
    auto* const kernel = attention_tiles_kernel<kDim, kFormat, kLoaderWarps, kBlocks>;
    const cudaError_t error = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (error != cudaSuccess) return error;
    uint32_t blocks = 0;
    for (uint32_t i = 0; i < params.a.pass_count; ++i) blocks += params.a.pass[i].tiles * params.a.pass[i].splits;
    return launch_behind(kernel, blocks, 32 * (kSoftmaxWarps + 1 + kLoaderWarps), bytes, stream, early_launch, params);
}

}  // namespace

cudaError_t launch_attention_tiles(const AttentionParams& params, const AttentionMaps& maps, KvFormat format, uint32_t* error_word,
                                   long long wait_limit_cycles, cudaStream_t stream, bool early_launch) {
    const TileParams tile_params{params, maps, error_word, wait_limit_cycles};
    const auto run = [&](auto dim) {
        constexpr int kDim = decltype(dim)::value;
        switch (format) {
        case KV_E4M3: return launch_tiles<kDim, KV_E4M3>(tile_params, stream, early_launch);
        case KV_E5M2: return launch_tiles<kDim, KV_E5M2>(tile_params, stream, early_launch);
        case KV_INT8: return launch_tiles<kDim, KV_INT8>(tile_params, stream, early_launch);
        default: return launch_tiles<kDim, KV_F16>(tile_params, stream, early_launch);
        }
    };
    return params.dim <= 64 ? run(std::integral_constant<int, 64>{}) : run(std::integral_constant<int, 128>{});
}

}  // namespace sdxlq
