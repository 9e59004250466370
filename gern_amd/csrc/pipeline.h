// What the files of libgern_pipelines.so share: the state behind a pipeline
// handle, the calling thread's error message and the step from a composed
// program to a compiled one.  Internal to the library.
#pragma once

#include "gern/core/composable.h"
#include "gern/runtime/runner.h"
#include "gern_pipelines.h"

#include <cstdint>
#include <memory>
#include <string>
#include <vector>

struct gern_pipeline_s {
    enum Kind { BLUR, SOFTMAX, GEMM_F32, GEMM_BF16, QK_SOFTMAX, GEMM_SCHEDULE, PAGE_TABLE, CACHE_WRITE, CACHE_ATTENTION, MATVEC4 } kind;
    std::unique_ptr<gern::Runner> runner;  // null in compile-only mode
    std::unique_ptr<gern::Runner> exact;   // GEMM: the direct-to-LDS matrix-core kernel (rows of A in whole 16-byte pieces)
    std::unique_ptr<gern::Runner> tail;    // fp32 GEMM in overwrite mode: C += of the last K % 4 columns
    bool accumulate = true;                // GEMM: C += A * B (false: C = A * B)
    int create_flags = 0;
    std::string source;
    std::string kernel_name;
    std::string exact_source, exact_kernel_name;
    bool last_run_exact = false;
    // blur
    int64_t nx = 0, ny = 0, stride = 0;
    // softmax / qk
    int64_t ncol = 0;
    int64_t head_dim = 0;
    // qk on 256 x 256 tiles: the memory through which the workgroups of a row block exchange row statistics
    bool qk_tiles = false;
    void *qk_scratch = nullptr;
    // the exchange memory of the library (csrc/qk_no_alloc.hip) on this pipeline's GPU; null if it has none
    void *qk_shared_scratch = nullptr;
    bool qk_used_shared = false;      // a run went through qk_shared_scratch since the last gern_pipeline_faults
    bool qk_default_period = true;    // built with the tag period every user of the shared memory agrees on
    void *last_stream = nullptr;
    // paged cache / 4-bit weights (csrc/serving_pipelines.cpp): one program per variant, and which one the last
    // run used.  Variants share the pipeline's other members.
    struct Variant {
        std::unique_ptr<gern::Runner> runner;  // null in compile-only mode
        std::string source;
        std::string kernel_name;
    };
    std::vector<Variant> variants;
    size_t last_variant = 0;
    int device = 0;  // the GPU that was current at creation, where the programs are loaded
    int64_t page_size = 0, group = 0;
    uint32_t *fault_count = nullptr;  // one device word: slots and pages outside the cache (gern_pipeline_faults)
    // parameter names
    std::vector<std::string> names;
};

namespace gern_detail {

#define GERN_DETAIL __attribute__((visibility("hidden")))

// Sets the calling thread's error message and returns 1.
GERN_DETAIL int fail(const std::string &msg);
// fail() with libgern_hip's message behind `who`.
GERN_DETAIL int failHip(const std::string &who);
// GERN_EXPERIMENTS=1 lets the environment change what the pipelines are built from (extra compiler
// options, other band heights and wavefront counts): for measurements, never needed for results.
GERN_DETAIL bool experiments();
// Generates (and, unless compile-only, loads) the program.
GERN_DETAIL int finish(gern_pipeline_s *p, gern::Composable program, int flags, int min_waves_per_simd = 0, int xcd_band_rows = 0);

}  // namespace gern_detail
