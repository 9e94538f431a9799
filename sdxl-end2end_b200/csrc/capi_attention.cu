// C ABI of the attention operators: validation and dispatch of the cache's copies and of shared-prefix attention.

#include "attention.cuh"
#include "context.cuh"

#include <algorithm>
#include <array>
#include <cmath>
#include <string>

using namespace sdxlq;

namespace {

// The context's device is the current one while this lives.
class DeviceScope {
public:
    explicit DeviceScope(const sdxlq_context* ctx) {
        if (cudaGetDevice(&previous_) != cudaSuccess) return;
        changed_ = previous_ != ctx->device && cudaSetDevice(ctx->device) == cudaSuccess;
    }
    ~DeviceScope() {
        if (changed_) cudaSetDevice(previous_);
    }
    DeviceScope(const DeviceScope&) = delete;
    DeviceScope& operator=(const DeviceScope&) = delete;

private:
    int previous_ = 0;
    bool changed_ = false;
};

constexpr uint64_t kMaxExtent = 0x7FFFFFFFull;
constexpr uint64_t kMaxStride = uint64_t(1) << 40;       // elements: products with the extents of memory that exists stay within 63 bits

bool is_kv_type(int32_t dtype) { return is_fp8(dtype) || dtype == SDXLQ_INT8 || dtype == SDXLQ_FP16; }
uint64_t element_bytes(int32_t dtype) { return dtype == SDXLQ_FP16 ? 2 : 1; }
bool aligned16(const void* pointer) { return reinterpret_cast<uintptr_t>(pointer) % 16 == 0; }
bool strides_ok(uint64_t bytes, uint64_t a, uint64_t b, uint64_t c) {
    return a <= kMaxStride && b <= kMaxStride && c <= kMaxStride && a * bytes % 16 == 0 && b * bytes % 16 == 0 && c * bytes % 16 == 0;
}

// Whether writing one head of `dim` elements may write another: each stride, in rising order, has to pass over all that the
// smaller ones reach. (Layouts whose axes interleave without meeting are refused with the others.)
bool overlapping(uint64_t dim, std::array<uint64_t, 3> extent, std::array<uint64_t, 3> stride) {
    std::array<int, 3> axis{0, 1, 2};
    std::sort(axis.begin(), axis.end(), [&](int a, int b) { return stride[a] < stride[b]; });
    uint64_t reach = dim;
    for (int i : axis) {
        if (extent[i] <= 1) continue;
        if (stride[i] < reach) return true;
        // strides are at most 2^40 and extents below 2^31: past this, no other stride is large enough
        if (stride[i] > (uint64_t(1) << 62) / extent[i]) reach = ~uint64_t(0);
        else reach += stride[i] * (extent[i] - 1);
    }
    return false;
}

bool absent(const sdxlq_kv_cache& c) { return c.slots == 0; }

// The checks that every reader and writer of a cache makes.
int validate_cache(sdxlq_context* ctx, const sdxlq_kv_cache& c) {
    if (!is_kv_type(c.dtype)) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: expects FP16, INT8 or FP8 elements");
    // a cache without room for a token has no memory
    if (c.capacity != 0 && (c.k == nullptr || c.v == nullptr)) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: null keys or values");
    if (c.capacity != 0 && c.dtype != SDXLQ_FP16 && (c.k_scales == nullptr || c.v_scales == nullptr)) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: an 8-bit cache needs scales");
    }
    if (c.heads == 0 || c.head_dim == 0) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: no heads");
    if (c.slots > kMaxExtent || c.capacity > kMaxExtent || c.heads > kMaxExtent) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "kv cache: dimensions too large");
    }
    const uint64_t unit = c.dtype == SDXLQ_FP16 ? 8 : 16;
    if (c.head_dim % unit != 0 || c.head_dim > 128) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE,
                    "kv cache: heads of at most 128 elements, a multiple of 8 for FP16 and of 16 for 8-bit types");
    }
    if (!aligned16(c.k) || !aligned16(c.v) || !strides_ok(element_bytes(c.dtype), c.slot_stride, c.token_stride, c.head_stride)) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "kv cache: keys, values and their strides must be multiples of 16 bytes");
    }
    return SDXLQ_OK;
}

KvView view_of(const sdxlq_kv_cache& c, const int32_t* lengths) {
    const int64_t bytes = static_cast<int64_t>(element_bytes(c.dtype));
    KvView v{};
    v.k = static_cast<uint8_t*>(c.k);
    v.v = static_cast<uint8_t*>(c.v);
    v.k_scales = c.k_scales;
    v.v_scales = c.v_scales;
    v.lengths = lengths;
    v.slot_stride = static_cast<int64_t>(c.slot_stride) * bytes;
    v.token_stride = static_cast<int64_t>(c.token_stride) * bytes;
    v.head_stride = static_cast<int64_t>(c.head_stride) * bytes;
    v.slots = static_cast<uint32_t>(c.slots);
    v.capacity = static_cast<uint32_t>(c.capacity);
    return v;
}

bool early(const sdxlq_context* ctx) { return ctx->early_launch && !ctx->profiling; }

int copy_tokens(sdxlq_context* ctx, const sdxlq_kv_cache* cache, const sdxlq_kv_tokens* tokens, bool write) {
    if (cache == nullptr || tokens == nullptr) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: null descriptor");
    const sdxlq_kv_tokens& t = *tokens;
    if (t.rows == 0 || t.tokens == 0) return SDXLQ_OK;
    const int status = validate_cache(ctx, *cache);
    if (status != SDXLQ_OK) return status;
    if (t.k == nullptr || t.v == nullptr) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: null tokens");
    if (t.first_slot > cache->slots || t.rows > cache->slots - t.first_slot) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: more rows than slots");
    }
    if (t.tokens > kMaxExtent || t.start > kMaxExtent) return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "kv cache: dimensions too large");
    if (t.positions == nullptr && (t.start > cache->capacity || t.tokens > cache->capacity - t.start)) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: tokens behind the capacity");
    }
    if (!aligned16(t.k) || !aligned16(t.v) || !strides_ok(2, t.row_stride, t.token_stride, t.head_stride)) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "kv cache: tokens and their strides must be multiples of 16 bytes");
    }
    if (write ? overlapping(cache->head_dim, {t.rows, cache->capacity, cache->heads}, {cache->slot_stride, cache->token_stride, cache->head_stride})
              : overlapping(cache->head_dim, {t.rows, t.tokens, cache->heads}, {t.row_stride, t.token_stride, t.head_stride})) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "kv cache: what is written overlaps in memory");
    }
    KvCopyLaunch launch{};
    launch.cache = view_of(*cache, nullptr);
    launch.k = static_cast<__half*>(t.k);
    launch.v = static_cast<__half*>(t.v);
    launch.row_stride = static_cast<int64_t>(t.row_stride);
    launch.token_stride = static_cast<int64_t>(t.token_stride);
    launch.head_stride = static_cast<int64_t>(t.head_stride);
    launch.positions = t.positions;
    launch.counts = t.counts;
    launch.rows = static_cast<uint32_t>(t.rows);
    launch.tokens = static_cast<uint32_t>(t.tokens);
    launch.heads = static_cast<uint32_t>(cache->heads);
    launch.dim = static_cast<uint32_t>(cache->head_dim);
    launch.first_slot = static_cast<uint32_t>(t.first_slot);
    launch.start = static_cast<uint32_t>(t.start);
    launch.format = static_cast<uint32_t>(cache->dtype);
    const DeviceScope device(ctx);
    LaunchTimer timer(ctx, SDXLQ_KERNEL_HARNESS);
    const cudaError_t error = write ? launch_kv_write(launch, ctx->stream, early(ctx)) : launch_kv_read(launch, ctx->stream, early(ctx));
    if (error == cudaErrorInvalidConfiguration) return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "kv cache: too many vectors for one call");
    if (error != cudaSuccess) return fail_cuda(ctx, error, "kv cache launch");
    return SDXLQ_OK;
}

uint64_t ceil_div(uint64_t a, uint64_t b) { return a / b + (a % b != 0); }

// Rows of a tile of the kernel that takes passes of so many rows: attention_rows.cu's with 16 or (heads of up to 64) 32, or
// attention_tiles.cu's with 128.
constexpr uint32_t kTensorTile = 128;
uint32_t row_tile_for(uint64_t rows, uint32_t dim, bool tensor) {
    if (tensor && rows > 32) return kTensorTile;
    return rows > 16 && dim <= 64 ? 32 : 16;
}

// Whether tensor maps can describe a part's strides. An extent of 1 may have any.
bool describable(const sdxlq_kv_cache& c) {
    const uint64_t extent[3] = {c.heads, c.capacity, c.slots}, stride[3] = {c.head_stride, c.token_stride, c.slot_stride};
    for (int axis = 0; axis < 3; ++axis) {
        if (extent[axis] > 1 && (stride[axis] == 0 || stride[axis] * 2 >= uint64_t(1) << 40)) return false;
    }
    return true;
}

// A call's passes, and what its launches need.
struct AttentionPlan {
    AttentionParams params{};
    KvFormat format[2] = {KV_F16, KV_F16};       // of each pass
    uint32_t row_tile[2] = {};
    uint64_t scratch_bytes = 0;
};

int plan_attention(sdxlq_context* ctx, int sm_count, const sdxlq_attention_desc& d, AttentionPlan& plan) {
    if (d.q == nullptr || d.y == nullptr) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: null query or output pointer");
    if (d.q_heads == 0 || d.head_dim == 0) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: no heads");
    if (d.batch > kMaxExtent || d.q_tokens > kMaxExtent || d.q_heads > kMaxExtent || d.batch * d.q_tokens > kMaxExtent ||
        d.batch * d.q_tokens * d.q_heads > kMaxExtent) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "attention: dimensions too large");
    }
    if (d.head_dim % 8 != 0 || d.head_dim > 128) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "attention: heads of at most 128 elements, a multiple of 8");
    }
    if (!aligned16(d.q) || !aligned16(d.y) || !strides_ok(2, d.q_batch_stride, d.q_token_stride, d.q_head_stride) ||
        !strides_ok(2, d.y_batch_stride, d.y_token_stride, d.y_head_stride)) {
        return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "attention: queries, outputs and their strides must be multiples of 16 bytes");
    }
    if (overlapping(d.head_dim, {d.batch, d.q_tokens, d.q_heads}, {d.y_batch_stride, d.y_token_stride, d.y_head_stride})) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: the output's rows overlap in memory");
    }
    if (!std::isfinite(d.scale)) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: the scale must be finite");
    const bool with_prefix = !absent(d.prefix), with_own = !absent(d.own);
    if (!with_prefix && !with_own) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: neither a prefix nor keys of its own");
    for (const sdxlq_kv_cache* part : {with_prefix ? &d.prefix : nullptr, with_own ? &d.own : nullptr}) {
        if (part == nullptr) continue;
        const int status = validate_cache(ctx, *part);
        if (status != SDXLQ_OK) return status;
        if (part->head_dim != d.head_dim) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: queries and keys differ in head size");
        if (d.q_heads % part->heads != 0) {
            return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: query heads must be a multiple of key heads");
        }
    }
    if (with_prefix && with_own && d.prefix.heads != d.own.heads) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: prefix and own keys differ in heads");
    }
    if (with_own && d.own.slots != d.batch) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: own keys must have a slot per batch entry");
    if (with_prefix && d.batch % d.prefix.slots != 0) {
        return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: the batch must be a multiple of the prefixes");
    }

    AttentionParams& p = plan.params;
    p.q = static_cast<const __half*>(d.q);
    p.y = static_cast<__half*>(d.y);
    p.q_batch = static_cast<int64_t>(d.q_batch_stride);
    p.q_token = static_cast<int64_t>(d.q_token_stride);
    p.q_head = static_cast<int64_t>(d.q_head_stride);
    p.y_batch = static_cast<int64_t>(d.y_batch_stride);
    p.y_token = static_cast<int64_t>(d.y_token_stride);
    p.y_head = static_cast<int64_t>(d.y_head_stride);
    if (with_prefix) p.prefix = view_of(d.prefix, d.prefix_lengths);
    if (with_own) p.own = view_of(d.own, d.own_lengths);
    p.batch = static_cast<uint32_t>(d.batch);
    p.q_tokens = static_cast<uint32_t>(d.q_tokens);
    p.q_heads = static_cast<uint32_t>(d.q_heads);
    p.kv_heads = static_cast<uint32_t>(with_prefix ? d.prefix.heads : d.own.heads);
    p.repeat = p.q_heads / p.kv_heads;
    p.dim = static_cast<uint32_t>(d.head_dim);
    p.rows_per_prefix = with_prefix ? p.batch / static_cast<uint32_t>(d.prefix.slots) : 1u;
    p.causal = d.causal != 0 ? 1u : 0u;
    p.scale_log2 = d.scale * 1.4426950408889634f;
    if (d.batch == 0 || d.q_tokens == 0) return SDXLQ_OK;

    const uint64_t entry_rows = static_cast<uint64_t>(p.q_tokens) * p.repeat;
    // Rows of the entries that share a prefix are taken together over it where that saves more than the join of the two
    // parts costs, which is about the time of four tiles of 128 keys for every tile of rows; a part that is of another
    // type has to be a pass of its own.
    const bool tensor = (!with_prefix || d.prefix.dtype != SDXLQ_FP16 || describable(d.prefix)) &&
                        (!with_own || d.own.dtype != SDXLQ_FP16 || describable(d.own));
    bool fold = false;
    if (with_prefix) {
        const uint64_t rows = entry_rows * p.rows_per_prefix;
        const uint64_t together = ceil_div(rows, row_tile_for(rows, p.dim, tensor));
        const uint64_t apart = p.rows_per_prefix * ceil_div(entry_rows, row_tile_for(entry_rows, p.dim, tensor));
        fold = (with_own && d.prefix.dtype != d.own.dtype) ||
               (together < apart && (!with_own || (apart - together) * ceil_div(p.prefix.capacity, 128) > 4 * apart));
    }
    const auto add_pass = [&](uint32_t members, bool prefix, bool own) {
        AttentionPass& pass = p.pass[p.pass_count];
        pass.members = members;
        pass.groups = p.batch / members;
        pass.rows = static_cast<uint32_t>(members * entry_rows);
        plan.format[p.pass_count] = static_cast<KvFormat>(prefix ? d.prefix.dtype : d.own.dtype);
        plan.row_tile[p.pass_count] = row_tile_for(pass.rows, p.dim, tensor);
        pass.row_tiles = static_cast<uint32_t>(ceil_div(pass.rows, plan.row_tile[p.pass_count++]));
        pass.with_prefix = prefix ? 1u : 0u;
        pass.with_own = own ? 1u : 0u;
    };
    if (fold) {
        add_pass(p.rows_per_prefix, true, false);
        if (with_own) add_pass(1, false, true);
    } else {
        add_pass(1, with_prefix, with_own);
    }
    p.by_row = p.pass_count > 1 ? 1u : 0u;
    uint64_t keys[2] = {}, work[2] = {};
    for (uint32_t i = 0; i < p.pass_count; ++i) {
        AttentionPass& pass = p.pass[i];
        const uint64_t tiles = static_cast<uint64_t>(pass.row_tiles) * p.kv_heads * pass.groups;
        if (tiles > kMaxExtent / 512) return fail(ctx, SDXLQ_ERR_UNSUPPORTED_SHAPE, "attention: dimensions too large");
        keys[i] = (pass.with_prefix ? p.prefix.capacity : 0ull) + (pass.with_own ? p.own.capacity : 0ull);
        pass.tiles = static_cast<uint32_t>(tiles);
        pass.splits = 1;
        work[i] = tiles * keys[i];
    }
    const bool one_launch = p.pass_count > 1 && plan.format[0] == plan.format[1] && plan.row_tile[0] == plan.row_tile[1];
    const uint32_t tensor_blocks = tile_blocks_per_sm(p.dim, plan.format[0]) * static_cast<uint32_t>(sm_count);
    if (p.pass_count == 1 && plan.row_tile[0] == kTensorTile) {
        // Blocks of like length come in waves of `tensor_blocks`. The tiles of the last wave, where it is not full, become a
        // pass of their own whose keys are split: `splits` shares of no less than 256 keys make ceil(rest * splits / tensor_blocks)
        // waves of 1 / splits the length. A wave also has about four key tiles' time of setting up and storing, and the join
        // as much again.
        const uint32_t tiles = p.pass[0].tiles, rest = tiles % tensor_blocks;
        const double key_tiles = static_cast<double>(keys[0]) / kTileKeys;
        uint32_t splits = 1;
        double least = key_tiles + 4.0;
        for (uint32_t s = 2; rest != 0 && s <= 64 && keys[0] / s >= 256; ++s) {
            const double time = static_cast<double>(ceil_div(static_cast<uint64_t>(rest) * s, tensor_blocks)) * (key_tiles / s + 4.0) + 4.0;
            if (time < least) {
                least = time;
                splits = s;
            }
        }
        if (splits > 1) {
            const uint32_t last = rest == tiles ? 0u : 1u;
            if (last == 1) {
                p.pass[1] = p.pass[0];
                plan.format[1] = plan.format[0];
                plan.row_tile[1] = plan.row_tile[0];
                p.pass[0].tiles = tiles - rest;
                p.pass_count = 2;
            }
            p.pass[last].first_tile = tiles - rest;
            p.pass[last].tiles = rest;
            p.pass[last].splits = splits;
        }
    } else {
        // The keys are split so that the blocks of a launch are of like size and fill the SMs once (tensor memory) or come to
        // about three per SM, none of less than 256 keys.
        for (uint32_t i = 0; i < p.pass_count; ++i) {
            const uint64_t blocks = plan.row_tile[i] == kTensorTile ? tile_blocks_per_sm(p.dim, plan.format[i]) * static_cast<uint64_t>(sm_count)
                                                                    : 3ull * sm_count;
            const uint64_t share = std::max<uint64_t>(256, ceil_div(one_launch ? work[0] + work[1] : work[i], blocks));
            p.pass[i].splits = static_cast<uint32_t>(std::clamp<uint64_t>(keys[i] / share, 1, 256));
        }
    }
    p.slots = 0;
    p.by_q_tokens.set(p.q_tokens);
    p.by_repeat.set(p.repeat);
    p.by_kv_heads.set(p.kv_heads);
    p.by_rows_per_prefix.set(p.rows_per_prefix);
    for (uint32_t i = 0; i < p.pass_count; ++i) {
        p.pass[i].by_tiles.set(p.pass[i].tiles);
        p.pass[i].by_row_tiles.set(p.pass[i].row_tiles);
        p.pass[i].first_slot = p.slots;
        p.slots = p.by_row ? p.slots + p.pass[i].splits : std::max(p.slots, p.pass[i].splits);
        if (!p.by_row && p.pass[i].splits > 1) p.slot_rows = static_cast<uint64_t>(p.pass[i].tiles) * plan.row_tile[i];
    }
    if (p.by_row) p.slot_rows = static_cast<uint64_t>(p.batch) * p.q_tokens * p.q_heads;
    if (p.slots > 1) plan.scratch_bytes = p.slots * p.slot_rows * (p.dim + 2) * sizeof(float);
    return SDXLQ_OK;
}

// The FP16 parts' tensor maps.
bool encode_maps(const sdxlq_context* ctx, const sdxlq_attention_desc& d, AttentionMaps& maps) {
    for (int i = 0; i < 2; ++i) {
        const sdxlq_kv_cache& c = i == 0 ? d.prefix : d.own;
        if (absent(c) || c.dtype != SDXLQ_FP16 || c.capacity == 0) continue;
        const cuuint64_t extent[4] = {c.head_dim, c.heads, c.capacity, c.slots};
        const uint64_t stride[3] = {c.head_stride, c.token_stride, c.slot_stride};
        cuuint64_t bytes[3];
        for (int axis = 0; axis < 3; ++axis) bytes[axis] = extent[axis + 1] == 1 ? 16 : stride[axis] * 2;
        const cuuint32_t box[4] = {64, 1, kTileKeys, 1}, step[4] = {1, 1, 1, 1};
        for (int part = 0; part < 2; ++part) {
            if (ctx->encode(&maps.map[i][part], CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, part == 0 ? c.k : c.v, extent, bytes, box, step,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS) {
                return false;
            }
        }
    }
    return true;
}

int run_attention(sdxlq_context* ctx, const sdxlq_attention_desc* desc) {
    if (desc == nullptr) return fail(ctx, SDXLQ_ERR_INVALID_ARGUMENT, "attention: null descriptor");
    const sdxlq_attention_desc& d = *desc;
    if (d.batch == 0 || d.q_tokens == 0) return SDXLQ_OK;
    AttentionPlan plan;
    int status = plan_attention(ctx, ctx->sm_count, d, plan);
    if (status != SDXLQ_OK) return status;
    AttentionParams& p = plan.params;
    if (p.slots > 1) {
        void* const scratch = d.scratch != nullptr ? d.scratch : ctx->workspace;
        const uint64_t room = d.scratch != nullptr ? d.scratch_bytes : ctx->workspace_bytes;
        if (plan.scratch_bytes > room || !aligned16(scratch)) {
            return fail(ctx, SDXLQ_ERR_WORKSPACE, "attention: needs " + std::to_string(plan.scratch_bytes) + " bytes of 16-byte aligned scratch");
        }
        p.part_o = static_cast<float*>(scratch);
        p.part_lse = reinterpret_cast<float2*>(p.part_o + p.slots * p.slot_rows * p.dim);
    }
    const DeviceScope device(ctx);
    const bool one_launch = p.pass_count == 1 || (plan.format[0] == plan.format[1] && plan.row_tile[0] == plan.row_tile[1]);
    LaunchTimer timer(ctx, SDXLQ_KERNEL_HARNESS, (one_launch ? 1 : 2) + (p.slots > 1 ? 1 : 0));
    cudaError_t error = cudaSuccess;
    AttentionMaps maps{};
    if ((plan.row_tile[0] == kTensorTile || plan.row_tile[1] == kTensorTile) && !encode_maps(ctx, d, maps)) {
        return fail(ctx, SDXLQ_ERR_CUDA, "attention: the driver refused a tensor map");
    }
    const auto launch = [&](const AttentionParams& params, uint32_t pass) {
        if (error != cudaSuccess) return;
        error = plan.row_tile[pass] == kTensorTile
                    ? launch_attention_tiles(params, maps, plan.format[pass], ctx->control, ctx->wait_limit_cycles, ctx->stream, early(ctx))
                    : launch_attention_rows(params, plan.format[pass], plan.row_tile[pass], ctx->stream, early(ctx));
    };
    if (one_launch) {
        launch(p, 0);
    } else {
        for (uint32_t i = 0; i < 2; ++i) {
            AttentionParams one = p;
            one.pass_count = 1;
            one.pass[0] = p.pass[i];
            launch(one, i);
        }
    }
    if (error == cudaSuccess && p.slots > 1) error = launch_attention_join(p, plan.row_tile[0], ctx->stream);
    if (error != cudaSuccess) return fail_cuda(ctx, error, "attention launch");
    return SDXLQ_OK;
}

}  // namespace

extern "C" {

int sdxlq_kv_cache_write(sdxlq_context* ctx, const sdxlq_kv_cache* cache, const sdxlq_kv_tokens* tokens) {
    if (ctx == nullptr) return SDXLQ_ERR_INVALID_ARGUMENT;
    try {
        return copy_tokens(ctx, cache, tokens, true);
    } catch (...) {
        return SDXLQ_ERR_CUDA;
    }
}

int sdxlq_kv_cache_read(sdxlq_context* ctx, const sdxlq_kv_cache* cache, const sdxlq_kv_tokens* tokens) {
    if (ctx == nullptr) return SDXLQ_ERR_INVALID_ARGUMENT;
    try {
        return copy_tokens(ctx, cache, tokens, false);
    } catch (...) {
        return SDXLQ_ERR_CUDA;
    }
}

int sdxlq_shared_prefix_attention(sdxlq_context* ctx, const sdxlq_attention_desc* desc) {
    if (ctx == nullptr) return SDXLQ_ERR_INVALID_ARGUMENT;
    try {
        return run_attention(ctx, desc);
    } catch (...) {
        return SDXLQ_ERR_CUDA;
    }
}

size_t sdxlq_shared_prefix_attention_scratch(const sdxlq_context* ctx, const sdxlq_attention_desc* desc) {
    if (ctx == nullptr || desc == nullptr || desc->batch == 0 || desc->q_tokens == 0) return 0;
    try {
        AttentionPlan plan;
        return plan_attention(nullptr, ctx->sm_count, *desc, plan) == SDXLQ_OK ? static_cast<size_t>(plan.scratch_bytes) : 0;
    } catch (...) {
        return 0;
    }
}

}
