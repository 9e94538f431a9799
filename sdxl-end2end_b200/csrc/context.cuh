// The context behind the C ABI and what every entry point does with it: launch timing and error reports.
#pragma once

#include "../../include/sdxlq.h"

#include <cuda.h>
#include <cuda_runtime.h>

#include <string>
#include <utility>
#include <vector>

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

constexpr int kPairChosen = 2;

struct sdxlq_context {
    int device = 0;
    cudaStream_t stream = nullptr;
    uint8_t* workspace = nullptr;
    size_t workspace_bytes = 0;
    float* norm_partials = nullptr;           // kNormPartialFloats floats: partial sums of sdxlq_group_norm_nhwc
    uint32_t* control = nullptr;           // [0] error word; from word 64: kMaxFp8Jobs amax words, then kMaxFp8Jobs
                                           // reader counters of the FP8 quantiser (all zero between calls)
    int sm_count = 148;
    uint8_t* staging = nullptr;            // pinned host image of the tables of a one-shot grouped call
    size_t staging_bytes = 0;
    cudaEvent_t staging_event = nullptr;   // completion of the last upload from `staging`
    int geglu_tile_n = 0;                     // tuning: accumulator tile width of GEGLU projections in grouped launches
                                              // (0: cost model). 128 lets the MMA issuer run three tiles ahead of the
                                              // GEGLU epilogues but measured slower (operand traffic, per-tile costs).
    int pair_mode = kPairChosen;              // kPairChosen: where they measured faster (see pairs_pay); 0 never use
                                              // CTA pairs, 1 whenever possible, -1 for traffic-bound launches only
    long long wait_limit_cycles = 4000000000LL;
    int forced_tile_n = 0;
    EncodeTiledFn encode = nullptr;
    uint32_t grouped_quant_threads = 0;       // tuning: block size of the rotated / general INT8 quantisers in grouped
                                              // launches (0: chosen per launch, see choose_quantiser_block)
    bool early_launch = true;                 // GEMM grids start while the quantiser before them drains (programmatic
                                              // dependent launch); the kernel waits before reading what it wrote
    sdxlq_int8_stats stats{};
    std::string last_error = "";
    // Optional per-kernel timing: CUDA event pairs recorded around each launch on the stream.
    bool profiling = false;
    struct TimedLaunch { int kernel_class; cudaEvent_t start; cudaEvent_t stop; int launches; };
    std::vector<TimedLaunch> timed;
    std::vector<std::pair<cudaEvent_t, cudaEvent_t>> event_pool;
};

namespace {

// Records an event pair around the launches issued while it is alive (profiling mode only).
class LaunchTimer {
public:
    LaunchTimer(sdxlq_context* ctx, int kernel_class, int launches = 1) : ctx_(ctx) {
        if (!ctx_->profiling) return;
        std::pair<cudaEvent_t, cudaEvent_t> events{nullptr, nullptr};
        if (!ctx_->event_pool.empty()) {
            events = ctx_->event_pool.back();
            ctx_->event_pool.pop_back();
        } else if (cudaEventCreate(&events.first) != cudaSuccess || cudaEventCreate(&events.second) != cudaSuccess) {
            return;
        }
        entry_ = {kernel_class, events.first, events.second, launches};
        active_ = cudaEventRecord(entry_.start, ctx_->stream) == cudaSuccess;
    }
    ~LaunchTimer() {
        if (!active_) return;
        cudaEventRecord(entry_.stop, ctx_->stream);
        ctx_->timed.push_back(entry_);
    }
    LaunchTimer(const LaunchTimer&) = delete;
    LaunchTimer& operator=(const LaunchTimer&) = delete;

private:
    sdxlq_context* ctx_;
    sdxlq_context::TimedLaunch entry_{};
    bool active_ = false;
};

int fail(sdxlq_context* ctx, int status, const std::string& message) {
    if (ctx != nullptr) ctx->last_error = message;
    return status;
}

int fail_cuda(sdxlq_context* ctx, cudaError_t error, const char* where) {
    return fail(ctx, SDXLQ_ERR_CUDA, std::string(where) + ": " + cudaGetErrorString(error));
}

bool is_fp8(int32_t dtype) { return dtype == SDXLQ_FP8_E4M3 || dtype == SDXLQ_FP8_E5M2; }

}  // namespace
