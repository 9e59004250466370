// C ABI over the operators of a serving step (include/gern_pipelines.h): block
// tables, the paged 8-bit cache of keys and values, attention over it, and
// products with 4-bit weights.  Like the other pipelines these are programs
// against Gern's C++ API; each launch is one gernel whose pieces are tiled over
// the grid.
#include "pipeline.h"

#include "annot/matvec4.h"
#include "annot/paged_cache.h"
#include "csrc/memory_ranges.h"
#include "gern_hip.h"

#include <algorithm>
#include <cstdint>
#include <iterator>

using namespace gern;
using gern_detail::fail;
using gern_detail::failHip;
using gern_detail::finish;
using gern_detail::overlap;
using gern_detail::Rows;

namespace {

// A pipeline under construction: destroyed unless it is handed out.
class Draft {
public:
    Draft(gern_pipeline_s::Kind kind, int flags) : p(new gern_pipeline_s{}), compile_only((flags & GERN_PIPELINE_COMPILE_ONLY) != 0) {
        p->kind = kind;
        p->create_flags = flags;
    }
    ~Draft() {
        if (p != nullptr) {
            gern_pipeline_destroy(p);
        }
    }
    Draft(const Draft &) = delete;
    Draft &operator=(const Draft &) = delete;
    gern_pipeline_s *operator->() {
        return p;
    }
    // Compiles one more program of the pipeline.
    int add(Composable program, int flags, int min_waves_per_simd = 0) {
        gern_pipeline_s one{};
        const int rc = finish(&one, program, flags, min_waves_per_simd);
        if (rc == 0) {
            const std::string name = one.runner ? one.runner->getKernelName() : one.kernel_name;
            p->variants.push_back({std::move(one.runner), one.source, name});
        }
        if (rc == 0 && !compile_only && gern_hip_current_device(&p->device) != 0) {
            return failHip("gern_hip_current_device");
        }
        return rc;
    }
    // The device word that gern_pipeline_faults reads.
    int addFaultCount(const char *who) {
        void *word = nullptr;
        if (compile_only) {
            return 0;
        }
        if (gern_hip_malloc(&word, sizeof(uint32_t)) != 0 || gern_hip_memset(word, 0, sizeof(uint32_t)) != 0) {
            if (word != nullptr) {
                gern_hip_free(word);
            }
            return failHip(who);
        }
        p->fault_count = static_cast<uint32_t *>(word);
        return 0;
    }
    gern_pipeline handOut() {
        gern_pipeline_s *done = p;
        p = nullptr;
        return done;
    }

private:
    gern_pipeline_s *p;
    bool compile_only;
};

bool usable(gern_pipeline p, gern_pipeline_s::Kind kind) {
    return p != nullptr && p->kind == kind;
}

bool compileOnly(gern_pipeline p) {
    return p->variants[0].runner == nullptr;
}

int evaluate(gern_pipeline p, size_t variant, const char *who, void *stream, const std::map<std::string, void *> &args) {
    try {
        Runner *runner = p->variants[variant].runner.get();
        if (runner == nullptr) {
            return fail(std::string(who) + ": the pipeline was created compile-only");
        }
        int device = -1;
        if (gern_hip_current_device(&device) != 0) {
            return failHip(who);
        }
        if (device != p->device) {
            return fail(std::string(who) + ": the pipeline was created on GPU " + std::to_string(p->device) + ", and GPU " + std::to_string(device) +
                        " is current");
        }
        runner->setStream(stream);
        runner->evaluate(args);
        p->last_variant = variant;
    } catch (const std::exception &e) {
        return fail(e.what());
    }
    return 0;
}

bool aligned(const void *pointer, uintptr_t bytes) {
    return reinterpret_cast<uintptr_t>(pointer) % bytes == 0;
}

struct Buffer {
    const void *at;
    int64_t bytes;
};

// A launch has less than 2^32 threads along x.
bool tooWide(int64_t workgroups, int64_t threads) {
    return workgroups * threads > 0xffffffff;
}

bool goodPageSize(int64_t page_size) {
    return page_size >= 16 && page_size <= 128 && (page_size & (page_size - 1)) == 0;
}

bool goodHeadDim(int64_t head_dim) {
    return head_dim >= 64 && head_dim <= 256 && head_dim % 64 == 0;
}

bool goodType(int type) {
    return type == GERN_TYPE_BF16 || type == GERN_TYPE_F16;
}

std::string typeName(int type) {
    return type == GERN_TYPE_BF16 ? "gernels::Bf16" : "gernels::F16";
}

// A name's Variable bound to a value, for PieceFunction's constants.
std::pair<const std::string, Variable> constant(const std::string &name, int64_t value) {
    return {name, Variable(name).bind(value)};
}

}  // namespace

extern "C" {

// --------------------------------------------------------------------------------------------- block tables

// Most requests a workgroup of 1024 threads takes the prefix sums of: eight a thread.
static_assert(GERN_PAGE_TABLE_MAX_REQUESTS == 8 * 1024, "the variants of gern_page_table_create");

int gern_page_table_create(int64_t page_size, int flags, gern_pipeline *out) {
    if (out == nullptr) {
        return fail("gern_page_table_create: null argument");
    }
    *out = nullptr;
    if (!goodPageSize(page_size)) {
        return fail("gern_page_table_create: page_size must be 16, 32, 64 or 128");
    }
    try {
        Draft p(gern_pipeline_s::PAGE_TABLE, flags);
        p->page_size = page_size;
        for (int64_t per : {1, 8}) {
            AbstractDataTypePtr batch(new const annot::WholeADT("batch", "gernels::RequestLengths"));
            AbstractDataTypePtr free_pages(new const annot::WholeADT("free_pages", "gernels::FreePages"));
            AbstractDataTypePtr table(
                new const annot::PiecesADT<hip::PageTableOut>("table", "gernels::PageTableOut", "share", {{"shares", &hip::PageTableOut::shares}}));
            annot::PieceFunction extend("gernels::extend_page_table", "gernels/serving/page_table.h", {batch, free_pages}, table, {"shares"},
                                        {"page", "threads", "per"});
            Variable one("one"), threads("block");
            Composable program = Global((Tile(table["shares"], one.bind(1)) || Grid::BLOCK_X)(
                                            extend[{constant("page", page_size), constant("threads", 1024), constant("per", per)}](batch, free_pages, table)),
                                        {{Grid::BLOCK_DIM_X, threads.bind(1024)}});
            if (p.add(program, flags | GERN_PIPELINE_NO_XCD_REMAP) != 0) {
                return 1;
            }
        }
        *out = p.handOut();
    } catch (const std::exception &e) {
        return fail(e.what());
    }
    return 0;
}

int gern_page_table_run(gern_pipeline p, const int32_t *cached, const int32_t *added, int64_t requests, const int32_t *free_pages,
                        int64_t free_capacity, const int32_t *free_count, int32_t *table, int64_t table_width, int32_t *lengths,
                        int32_t *starts, int32_t *slots, int64_t tokens, int32_t *counts, void *stream) {
    if (!usable(p, gern_pipeline_s::PAGE_TABLE)) {
        return fail("gern_page_table_run: bad pipeline");
    }
    if (requests < 0 || requests > GERN_PAGE_TABLE_MAX_REQUESTS) {
        return fail("gern_page_table_run: requests must be in [0, GERN_PAGE_TABLE_MAX_REQUESTS = 8192]");
    }
    if (table_width < 1 || table_width > 0x7fffffff || tokens < 0 || tokens > 0x7fffffff || free_capacity < 0 || free_capacity > 0x7fffffff) {
        return fail("gern_page_table_run: table_width must be in [1, 2^31), tokens and free_capacity in [0, 2^31)");
    }
    if (free_count == nullptr || starts == nullptr || counts == nullptr || (requests > 0 && (cached == nullptr || added == nullptr || table == nullptr || lengths == nullptr)) ||
        (tokens > 0 && slots == nullptr) || (free_capacity > 0 && free_pages == nullptr)) {
        return fail("gern_page_table_run: null buffer");
    }
    const Buffer in[] = {{cached, 4 * requests}, {added, 4 * requests}, {free_pages, 4 * free_capacity}, {free_count, 4}};
    const Buffer results[] = {{table, 4 * requests * table_width}, {lengths, 4 * requests}, {starts, 4 * (requests + 1)}, {slots, 4 * tokens}, {counts, 8}};
    for (const auto &b : in) {
        if (!aligned(b.at, 4)) {
            return fail("gern_page_table_run: buffers must be 4-byte aligned");
        }
    }
    for (const auto &r : results) {
        if (!aligned(r.at, 4)) {
            return fail("gern_page_table_run: buffers must be 4-byte aligned");
        }
        for (const auto &b : in) {
            if (overlap(r.at, r.bytes, b.at, b.bytes)) {
                return fail("gern_page_table_run: a result shares memory with an input (workgroups read the inputs while others write)");
            }
        }
        for (const auto &other : results) {
            if (&other != &r && overlap(r.at, r.bytes, other.at, other.bytes)) {
                return fail("gern_page_table_run: two results share memory");
            }
        }
    }
    hip::RequestLengths batch{cached, added, requests};
    hip::FreePages list{free_pages, free_count, free_capacity};
    // a workgroup for every 1024 tokens of the slot map, at most one for each CU
    const int64_t shares = std::clamp<int64_t>((tokens + 1023) / 1024, 1, 256);
    hip::PageTableOut result{table, lengths, starts, slots, counts, table_width, tokens, shares};
    return evaluate(p, requests <= 1024 ? 0 : 1, "gern_page_table_run", stream, {{"batch", &batch}, {"free_pages", &list}, {"table", &result}});
}

// --------------------------------------------------------------------------------------------- writing the cache

namespace {

// Checks of a cache that every operator over it makes; empty when it is fine.
std::string cacheProblem(const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, int64_t pages, int64_t heads,
                         int64_t page_size) {
    if (k_cache == nullptr || v_cache == nullptr || k_scales == nullptr || v_scales == nullptr) {
        return "null cache";
    }
    if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k_scales, 4) || !aligned(v_scales, 4)) {
        return "the cache's codes must be 16-byte aligned and its scales 4-byte aligned";
    }
    if (heads < 1 || heads > 65535) {
        return "heads must be in [1, 65535]";
    }
    if (pages < 1 || pages > 0x7fffffff / page_size) {
        return "pages must be at least 1, and pages * page_size less than 2^31";
    }
    return "";
}

struct CacheBuffers {
    Buffer codes[2], scales[2];
};
CacheBuffers cacheBuffers(gern_pipeline p, const void *k_cache, const void *v_cache, const float *k_scales, const float *v_scales, int64_t pages,
                          int64_t heads) {
    const int64_t scales = pages * heads * (int64_t)sizeof(float), codes = pages * heads * p->page_size * p->head_dim;
    return {{{k_cache, codes}, {v_cache, codes}}, {{k_scales, scales}, {v_scales, scales}}};
}

}  // namespace

int gern_cache_write_create(int64_t head_dim, int64_t page_size, int type, int flags, gern_pipeline *out) {
    if (out == nullptr) {
        return fail("gern_cache_write_create: null argument");
    }
    *out = nullptr;
    if (!goodHeadDim(head_dim) || !goodPageSize(page_size) || !goodType(type)) {
        return fail("gern_cache_write_create: head_dim must be 64, 128, 192 or 256, page_size 16, 32, 64 or 128, and type GERN_TYPE_BF16 or "
                    "GERN_TYPE_F16");
    }
    try {
        Draft p(gern_pipeline_s::CACHE_WRITE, flags);
        p->head_dim = head_dim;
        p->page_size = page_size;
        for (int64_t threads : {64, 256}) {
            AbstractDataTypePtr tokens(new const annot::WholeADT("tokens", "gernels::NewTokensOf<" + typeName(type) + ">"));
            using Cache = hip::WritableCache;
            AbstractDataTypePtr cache(new const annot::PiecesADT<Cache>("cache", "gernels::WritableCache", "at", {{"pieces", &Cache::pieces}}));
            annot::PieceFunction write("gernels::write_cache", "gernels/serving/cache_write.h", {tokens}, cache, {"pieces"}, {"head_dim", "page", "threads"});
            Variable x("x"), block("block");
            Composable program = Global((Tile(cache["pieces"], x.bind(1)) || Grid::BLOCK_X)(write[{constant("head_dim", head_dim), constant("page", page_size),
                                                                                                   constant("threads", threads)}](tokens, cache)),
                                        {{Grid::BLOCK_DIM_X, block.bind(threads)}});
            if (p.add(program, flags | GERN_PIPELINE_NO_XCD_REMAP) != 0) {
                return 1;
            }
        }
        if (p.addFaultCount("gern_cache_write_create") != 0) {
            return 1;
        }
        *out = p.handOut();
    } catch (const std::exception &e) {
        return fail(e.what());
    }
    return 0;
}

int gern_cache_write_run(gern_pipeline p, const void *K, int64_t ldk, const void *V, int64_t ldv, const int32_t *slots, int64_t tokens,
                         int64_t heads, uint8_t *k_cache, uint8_t *v_cache, float *k_scales, float *v_scales, int64_t pages, void *stream) {
    if (!usable(p, gern_pipeline_s::CACHE_WRITE)) {
        return fail("gern_cache_write_run: bad pipeline");
    }
    const std::string problem = cacheProblem(k_cache, v_cache, k_scales, v_scales, pages, heads, p->page_size);
    if (!problem.empty()) {
        return fail("gern_cache_write_run: " + problem);
    }
    if (tokens < 0 || tokens > 0x7fffffff) {
        return fail("gern_cache_write_run: tokens must be in [0, 2^31)");
    }
    if (tokens == 0) {
        return 0;
    }
    if (K == nullptr || V == nullptr || slots == nullptr) {
        return fail("gern_cache_write_run: null buffer");
    }
    if (!aligned(K, 16) || !aligned(V, 16) || ldk % 8 != 0 || ldv % 8 != 0 || !aligned(slots, 4)) {
        return fail("gern_cache_write_run: K and V are read in 16-byte pieces: both must be 16-byte aligned and their row strides multiples of 8 "
                    "elements (slots 4-byte aligned)");
    }
    if (ldk < heads * p->head_dim || ldv < heads * p->head_dim) {
        return fail("gern_cache_write_run: a row stride is less than heads * head_dim");
    }
    hip::NewTokens fresh{K, V, ldk / 2, ldv / 2, slots, tokens};
    // One token per workgroup of one wavefront while that gives no more workgroups than the GPU runs at a time;
    // beyond that a page's worth of tokens per workgroup of four.  us, 8 heads of 128, one / the other: 256 requests of one
    // token, pages of 16 8.4 / 18, of 128 8.5 / 183; 1024 requests 9.9 / 25, 11.5 / 183; a prompt of 8192 tokens 15.4 / 8.3,
    // 31 / 8.3.  A prompt of 1024 tokens, 8.5 / 8.6 and 16.2 / 8.4, looks like 1024 requests from here.
    const bool single = tokens * heads * 2 <= 16384;
    const int64_t stretch = single ? 1 : p->page_size;
    const int64_t pieces = (tokens + stretch - 1) / stretch * heads * 2;
    if (pieces > 0x7fffffff) {
        return fail("gern_cache_write_run: tokens / page_size * heads must be less than 2^30");
    }
    if (tooWide(pieces, single ? 64 : 256)) {
        return fail("gern_cache_write_run: tokens / page_size * heads must be less than 2^23");
    }
    if (!compileOnly(p)) {
        const CacheBuffers buffers = cacheBuffers(p, k_cache, v_cache, k_scales, v_scales, pages, heads);
        const Buffer results[] = {buffers.codes[0], buffers.codes[1], buffers.scales[0], buffers.scales[1]};
        const int64_t width = heads * p->head_dim * 2;
        for (const auto &r : results) {
            if (overlap(Rows{K, tokens, ldk * 2, width}, r.at, r.bytes) || overlap(Rows{V, tokens, ldv * 2, width}, r.at, r.bytes) ||
                overlap(slots, 4 * tokens, r.at, r.bytes)) {
                return fail("gern_cache_write_run: K, V or the slots share memory with the cache");
            }
            for (const auto &other : results) {
                if (&other != &r && overlap(r.at, r.bytes, other.at, other.bytes)) {
                    return fail("gern_cache_write_run: codes or scales of keys and of values share memory");
                }
            }
        }
    }
    hip::WritableCache cache{{k_cache, v_cache, k_scales, v_scales, pages, heads, p->fault_count}, pieces, stretch};
    return evaluate(p, single ? 0 : 1, "gern_cache_write_run", stream, {{"tokens", &fresh}, {"cache", &cache}});
}

// --------------------------------------------------------------------------------------------- attention

namespace {

// How a run divides its work: which program, and the split of the keys.
struct AttentionPlan {
    size_t variant;
    int64_t row_tiles, splits, chunk;
    bool whole_will_do;  // workgroups are enough without a split
};

constexpr int64_t kMaxSplits = 256;  // gernels/serving/cache_attention.h, join_splits

// The programs of a pipeline: few rows (queries times the heads that share a head of the cache) against keys that the
// wavefronts divide, many rows divided among the wavefronts, and few rows on twice the wavefronts where workgroups are few.
struct AttentionProgram {
    bool few;
    int64_t waves;
};
constexpr AttentionProgram kAttentionPrograms[] = {{true, 4}, {false, 4}, {true, 8}};
constexpr size_t kFewRows = 0, kManyRows = 1, kFewRowsWide = 2, kJoinWave = 3, kJoinWorkgroup = 4;

// 16-row tiles of a wavefront of the second: accumulators and queries take 3/8 R D registers a lane, and two
// wavefronts are to fit a SIMD.
int64_t attentionRowTiles(int64_t head_dim) {
    return head_dim <= 128 ? 2 : 1;
}

// Wavefronts of the first that its registers leave room for on a SIMD.
int attentionResidentWaves(int64_t head_dim) {
    return head_dim == 64 ? 4 : head_dim == 128 ? 3 : 2;
}

AttentionPlan attentionPlan(int64_t head_dim, int64_t requests, int64_t heads, int64_t rows, int64_t max_length) {
    AttentionPlan plan{};
    // us with the program for few / many rows: 32 requests of 2000 to 4000 keys, 8 heads, 16 rows of 64 dimensions 30 / 62, of
    // 128 44 / 93, of 192 60 / 103, of 256 91 / 114; 64 rows 59 / 68, 95 / 102, 117 / 116, 164 / 130; 96 rows 60 / 77, 100 / 113,
    // 113 / 153, 153 / 168; 128 rows 81 / 78, 121 / 115, 157 / 162, 205 / 177.  4 requests of 500 to 1000, 64 rows: 10 / 29,
    // 12 / 40, - , 18 / 41.
    plan.variant = rows <= 64 ? kFewRows : kManyRows;
    const int64_t tile = plan.variant == kFewRows ? 16 : 16 * kAttentionPrograms[kManyRows].waves * attentionRowTiles(head_dim);
    plan.row_tiles = std::max<int64_t>(1, (rows + tile - 1) / tile);
    // Keys are split, into pieces of at least 512, until there are `wanted` workgroups.  Eight for each of 256 CUs: two
    // to three times what is resident, so that requests of different lengths leave few CUs idle at the end.  Few rows of
    // more than 128 dimensions: two, what is resident, because the joined parts are larger and a start costs more (32
    // requests of 2000 to 4000 keys, 8 heads, one query, with 512 / 1024 / 2048: of 64 dimensions 28 / 26 / 28, of 128
    // 38 / 44 / 42, of 192 56 / 58 / 64, of 256 89 / 87 / 92; 2 of 65536 to 131072: 48 / 43 / 40, 84 / 77 / 79,
    // 114 / 121 / 116, 150 / 156 / 149).
    // Measured (us) with 512 / 1024 / 2048 / 4096: 64 requests of 4096 to 8192 keys, 8 heads of 128: 181 / 175 / 155 /
    // 165; 3 of 131072 to 262144: 266 / 188 / 184 / 197; 32 of 1250 to 2500, 16 heads of 256: 95 / 110 / 109 / -; 6 of 113
    // to 447 queries and 4032 to 5915 keys, 4 heads of 64 for 16: - / 103 / 97 / 103.
    const int64_t wanted = plan.variant == kFewRows && head_dim > 128 ? 512 : 2048;
    const int64_t whole = requests * heads * plan.row_tiles;
    // Up to 1024 keys are not worth a second launch (1 request of 1000, 8 heads of 128: 10.3 us whole, 11.9 split;
    // 2000: 16.0, 12.1), nor are workgroups for every CU four times over (128 requests of 1000 to 2000, 8 heads
    // of 128: 87 whole, 97 in two).  Pieces of 256 / 512 / 1024 at least: 16 requests of 2000 to 4000 33.3 / 31.7 / 27.5, one
    // of 32768 18.4 / 17.1 / 19.5, two of 20000, 4 heads 16.0 / 15.8 / 18.6.
    int64_t splits = max_length <= 1024 || whole >= 1024 ? 1 : std::clamp<int64_t>((wanted + whole - 1) / whole, 1, kMaxSplits);
    // But a request that is far longer than the others must not be what all wait for: few rows in workgroups enough are
    // divided into pieces of 4096 keys, as long as the parts of `rows` queries a request take no more than 256 MiB.  Whole /
    // pieces of 2048 / 4096 / 8192 (us, 8 heads of 128): 127 requests of 4000 to 8000 and one of 262144 3176 / 737 / 730 /
    // 809, one of 20000 388 / 322 / 315 / 345; 128 of 2000 to 4000 153 / 158 / - / -, of 4096 to 8192 312 / 302 / 294 / -,
    // of 16384 to 32768 1182 / 1112 / 1086 / 1088.
    plan.whole_will_do = plan.variant == kFewRows && whole >= 1024;
    if (plan.whole_will_do) {
        const int64_t part = requests * heads * rows * (head_dim + 2) * (int64_t)sizeof(float);
        splits = std::clamp<int64_t>(std::min<int64_t>((max_length + 4095) / 4096, (256 << 20) / part), 1, kMaxSplits);
    }
    // Undivided keys, and a CU for every workgroup: its wavefronts' steps of 32 keys one after the other are what a call
    // takes, so there are twice as many.  8 heads of 64, 128, 192, 256, us with 4 / 8 wavefronts: 1 request of 500 to 1000
    // keys 10.6 / 10.2, 12.3 / 10.9, 13.8 / 12.4, 16.7 / 16.0; 32 11.4 / 10.2, 15.5 / 13.9, 18.7 / 17.7, 21.8 / 23.5; 1 of 250 to
    // 500 10.6 / 10.5, 10.2 / 10.3, 10.1 / 10.1, 11.3 / 11.6; 64 of 1000, 128, two workgroups a CU, 24 / 26.
    if (plan.variant == kFewRows && max_length > 512 && max_length <= 1024 && whole <= 256) {
        plan.variant = kFewRowsWide;
    }
    plan.chunk = std::max<int64_t>(512, ((max_length + splits - 1) / splits + 255) / 256 * 256);
    plan.splits = std::max<int64_t>(1, (max_length + plan.chunk - 1) / plan.chunk);
    // BLOCK_Y holds 65535 pieces; a workgroup takes further row tiles in turn
    plan.row_tiles = std::min(plan.row_tiles, 65535 / plan.splits);
    return plan;
}

int64_t attentionWorkspace(const AttentionPlan &plan, int64_t tokens, int64_t q_heads, int64_t head_dim) {
    return plan.splits == 1 ? 0 : plan.splits * tokens * q_heads * (head_dim + 2) * (int64_t)sizeof(float);
}

// Checks of the sizes that a run and its workspace depend on; empty when they are fine.
std::string attentionProblem(int64_t tokens, int64_t requests, int64_t q_heads, int64_t heads, int64_t max_queries, int64_t max_length) {
    if (heads < 1 || heads > 65535 || q_heads < heads || q_heads % heads != 0) {
        return "heads must be in [1, 65535] and q_heads a multiple of it";
    }
    if (requests < 0 || requests > 65535) {
        return "requests must be in [0, 65535]";
    }
    if (tokens < 0 || max_queries < 1 || max_queries > 0x7fffffff / q_heads || tokens > 0x7fffffff / q_heads) {
        return "tokens * q_heads and max_queries * q_heads must be less than 2^31, and max_queries at least 1";
    }
    if (max_length < 1 || max_length > GERN_CACHE_MAX_LENGTH) {
        return "max_length must be in [1, GERN_CACHE_MAX_LENGTH]";
    }
    return "";
}

}  // namespace

int gern_cache_attention_create(int64_t head_dim, int64_t page_size, int type, int flags, gern_pipeline *out) {
    if (out == nullptr) {
        return fail("gern_cache_attention_create: null argument");
    }
    *out = nullptr;
    if (!goodHeadDim(head_dim) || !goodPageSize(page_size) || !goodType(type)) {
        return fail("gern_cache_attention_create: head_dim must be 64, 128, 192 or 256, page_size 16, 32, 64 or 128, and type GERN_TYPE_BF16 or "
                    "GERN_TYPE_F16");
    }
    try {
        Draft p(gern_pipeline_s::CACHE_ATTENTION, flags);
        p->head_dim = head_dim;
        p->page_size = page_size;
        const std::string header = "gernels/serving/cache_attention.h", batch_type = "gernels::AttentionBatchOf<" + typeName(type) + ">";
        AbstractDataTypePtr batch(new const annot::WholeADT("batch", batch_type));
        AbstractDataTypePtr cache(new const annot::WholeADT("cache", "gernels::PagedCache"));
        for (const AttentionProgram &attention : kAttentionPrograms) {
            const bool few = attention.few;
            using Out = hip::AttentionOut;
            AbstractDataTypePtr result(new const annot::PiecesADT<Out>("result", "gernels::AttentionOut", "piece",
                                                                      {{"pieces", &Out::pieces}, {"heads", &Out::heads}, {"requests", &Out::requests}}));
            const std::vector<std::string> constants = few ? std::vector<std::string>{"head_dim", "page", "waves"} :
                                                             std::vector<std::string>{"head_dim", "page", "row_tiles", "waves"};
            annot::PieceFunction attend(few ? "gernels::attend_few_rows" : "gernels::attend_many_rows", header, {batch, cache}, result,
                                        {"pieces", "heads", "requests"}, constants);
            std::map<std::string, Variable> bound{constant("head_dim", head_dim), constant("page", page_size), constant("waves", attention.waves)};
            if (!few) {
                bound.insert(constant("row_tiles", attentionRowTiles(head_dim)));
            }
            Variable x("x"), head("head"), request("request"), threads("threads");
            // Heads along BLOCK_X: the workgroups that run together read the heads of the same pages, which stand side by
            // side (3 requests of 131072 to 262144 keys: 222 us with the pieces of the keys along BLOCK_X, 188 so).
            Composable program = Global(
                (Tile(result["pieces"], x.bind(1)) || Grid::BLOCK_Y)((Tile(result["heads"], head.bind(1)) || Grid::BLOCK_X)(
                    (Tile(result["requests"], request.bind(1)) || Grid::BLOCK_Z)(attend[bound](batch, cache, result)))),
                {{Grid::BLOCK_DIM_X, threads.bind(64 * attention.waves)}});
            // wavefronts of the second program on a SIMD
            if (p.add(program, flags | GERN_PIPELINE_NO_XCD_REMAP, few ? attentionResidentWaves(head_dim) : head_dim == 64 ? 3 : 2) != 0) {
                return 1;
            }
        }
        using Rows = hip::JoinRows;
        for (int64_t per_row : {1, 4}) {
            AbstractDataTypePtr rows(new const annot::PiecesADT<Rows>("rows", "gernels::JoinRows", "block", {{"blocks", &Rows::blocks}}));
            annot::PieceFunction join("gernels::join_splits", header, {batch}, rows, {"blocks"}, {"head_dim", "waves", "per_row"});
            Variable x("x"), threads("threads");
            Composable program = Global((Tile(rows["blocks"], x.bind(1)) || Grid::BLOCK_X)(
                                            join[{constant("head_dim", head_dim), constant("waves", 4), constant("per_row", per_row)}](batch, rows)),
                                        {{Grid::BLOCK_DIM_X, threads.bind(256)}});
            if (p.add(program, flags | GERN_PIPELINE_NO_XCD_REMAP) != 0) {
                return 1;
            }
        }
        if (p.addFaultCount("gern_cache_attention_create") != 0) {
            return 1;
        }
        *out = p.handOut();
    } catch (const std::exception &e) {
        return fail(e.what());
    }
    return 0;
}

int gern_cache_attention_workspace(gern_pipeline p, int64_t tokens, int64_t requests, int64_t q_heads, int64_t heads, int64_t max_queries,
                                   int64_t max_length, int64_t *bytes) {
    if (!usable(p, gern_pipeline_s::CACHE_ATTENTION) || bytes == nullptr) {
        return fail("gern_cache_attention_workspace: bad pipeline or null argument");
    }
    const std::string problem = attentionProblem(tokens, requests, q_heads, heads, max_queries, max_length);
    if (!problem.empty()) {
        return fail("gern_cache_attention_workspace: " + problem);
    }
    *bytes = requests == 0 ? 0
                           : attentionWorkspace(attentionPlan(p->head_dim, requests, heads, max_queries * (q_heads / heads), max_length), tokens, q_heads,
                                                p->head_dim);
    return 0;
}

int gern_cache_attention_run(gern_pipeline p, const void *Q, int64_t ldq, const uint8_t *k_cache, const uint8_t *v_cache, const float *k_scales,
                             const float *v_scales, int64_t pages, const int32_t *table, int64_t table_width, const int32_t *lengths,
                             const int32_t *starts, int64_t requests, int64_t tokens, int64_t q_heads, int64_t heads, void *O, int64_t ldo,
                             float scale, int64_t max_queries, int64_t max_length, void *workspace, int64_t workspace_bytes, void *stream) {
    const char *who = "gern_cache_attention_run";
    if (!usable(p, gern_pipeline_s::CACHE_ATTENTION)) {
        return fail("gern_cache_attention_run: bad pipeline");
    }
    std::string problem = attentionProblem(tokens, requests, q_heads, heads, max_queries, max_length);
    if (problem.empty()) {
        problem = cacheProblem(k_cache, v_cache, k_scales, v_scales, pages, heads, p->page_size);
    }
    if (!problem.empty()) {
        return fail("gern_cache_attention_run: " + problem);
    }
    if (table_width < 1 || table_width > GERN_CACHE_MAX_LENGTH / p->page_size) {
        return fail("gern_cache_attention_run: table_width must be at least 1 and table_width * page_size at most GERN_CACHE_MAX_LENGTH");
    }
    if (requests == 0 || tokens == 0) {
        return 0;
    }
    if (Q == nullptr || O == nullptr || table == nullptr || lengths == nullptr || starts == nullptr) {
        return fail("gern_cache_attention_run: null buffer");
    }
    if (!aligned(Q, 16) || !aligned(O, 16) || ldq % 8 != 0 || ldo % 8 != 0 || !aligned(table, 4) || !aligned(lengths, 4) || !aligned(starts, 4)) {
        return fail("gern_cache_attention_run: Q and O are moved in 16-byte pieces: both must be 16-byte aligned and their row strides multiples of 8 "
                    "elements (table, lengths and starts 4-byte aligned)");
    }
    if (ldq < q_heads * p->head_dim || ldo < q_heads * p->head_dim) {
        return fail("gern_cache_attention_run: a row stride is less than q_heads * head_dim");
    }
    const int64_t group = q_heads / heads;
    AttentionPlan plan = attentionPlan(p->head_dim, requests, heads, max_queries * group, max_length);
    int64_t needed = attentionWorkspace(plan, tokens, q_heads, p->head_dim);
    if (plan.whole_will_do && (workspace == nullptr || workspace_bytes < needed || !aligned(workspace, 16))) {
        plan.splits = 1;
        needed = 0;
    }
    if (needed > 0 && (workspace == nullptr || workspace_bytes < needed || !aligned(workspace, 16))) {
        return fail("gern_cache_attention_run: the workspace must be 16-byte aligned and hold the " + std::to_string(needed) +
                    " bytes that gern_cache_attention_workspace says");
    }
    // one query, 8 heads of 128, us with a wavefront / a workgroup a row: 8 splits 13.7 / 13.6, 16 13.7 / 14.1, 32 13.9 / 14.6,
    // 63 19.0 / 17.4; 300 queries, 14 splits 97 / 101
    const bool wave_a_row = plan.splits <= 16;
    const int64_t rows = tokens * q_heads, join_blocks = wave_a_row ? (rows + 3) / 4 : rows;
    if (needed > 0 && tooWide(join_blocks, 256)) {
        return fail("gern_cache_attention_run: tokens * q_heads must be less than 2^24 where keys are split into more than 16 pieces, 2^26 into fewer");
    }
    const Rows q{Q, tokens, ldq * 2, q_heads * p->head_dim * 2}, o{O, tokens, ldo * 2, q_heads * p->head_dim * 2};
    if (needed > 0 && overlap(o, workspace, needed)) {
        return fail("gern_cache_attention_run: the workspace shares memory with O");
    }
    if (!compileOnly(p)) {
        const CacheBuffers buffers = cacheBuffers(p, k_cache, v_cache, k_scales, v_scales, pages, heads);
        const Buffer in[] = {buffers.codes[0], buffers.codes[1], buffers.scales[0], buffers.scales[1], {table, 4 * requests * table_width},
                             {lengths, 4 * requests}, {starts, 4 * (requests + 1)}};
        const bool in_place = Q == O && (ldq == ldo || tokens == 1);
        if (!in_place && overlap(q, o)) {
            return fail("gern_cache_attention_run: O shares memory with Q and is not in its place");
        }
        if (needed > 0 && overlap(q, workspace, needed)) {
            return fail("gern_cache_attention_run: the workspace shares memory with Q");
        }
        for (const auto &b : in) {
            if (overlap(o, b.at, b.bytes) || overlap(workspace, needed, b.at, b.bytes)) {
                return fail("gern_cache_attention_run: O or the workspace shares memory with the cache, the table, lengths or starts");
            }
        }
    }
    float *partial = static_cast<float *>(workspace), *stats = needed > 0 ? partial + plan.splits * rows * p->head_dim : nullptr;
    hip::AttentionBatch batch{Q, ldq / 2, table, lengths, starts, table_width, tokens, group, scale * 1.4426950408889634f};
    hip::PagedCache cache{const_cast<uint8_t *>(k_cache), const_cast<uint8_t *>(v_cache), const_cast<float *>(k_scales), const_cast<float *>(v_scales),
                          pages, heads, p->fault_count};
    hip::AttentionOut result{O, ldo / 2, partial, stats, plan.splits, plan.chunk, plan.row_tiles * plan.splits, heads, requests};
    const int rc = evaluate(p, plan.variant, who, stream, {{"batch", &batch}, {"cache", &cache}, {"result", &result}});
    if (rc != 0 || plan.splits == 1) {
        return rc;
    }
    hip::JoinRows join{O, ldo / 2, partial, stats, starts, plan.splits, requests, q_heads, rows, join_blocks};
    const int joined = evaluate(p, wave_a_row ? kJoinWave : kJoinWorkgroup, who, stream, {{"batch", &batch}, {"rows", &join}});
    p->last_variant = plan.variant;
    return joined;
}

// --------------------------------------------------------------------------------------------- 4-bit weights

namespace {

struct MatvecShape {
    int64_t row_tiles, column_tiles;
};
// The programs of a pipeline, by tiles of 16 rows (0: up to 4 rows) and of 16 columns; 8 wavefronts each.
constexpr MatvecShape kMatvecShapes[] = {{0, 1}, {0, 2}, {0, 4}, {1, 1}, {1, 2}, {1, 3}, {1, 4}, {2, 1}, {2, 4}, {4, 1}, {4, 4}};
constexpr int64_t kMatvecWaves = 8;

// The program for M rows and N columns: the one whose slowest CU has least to do, with a workgroup a CU at a time (more
// fit, and share what it can do).  A workgroup's work is its tiles of
// columns, and what it does for x whatever their number: as much as 0.7 of a tile with up to 4 rows, as 2 tiles for
// every 16 rows beyond that.  Measured (us, K = 8192 but where said), one to four tiles of columns:
//   1 row:   28672 columns 33 / 31 / 31 / 30, 16384 of K = 4096 9.7 / 9.8 / - / 9.2, 8192 11.3 / 9.7 / - / 12.5
//   13 rows: 10001 columns 27 / 24 / 16.6 / 18.7;  16 rows: 20000 - / - / 33 / 37, 32768 of K = 4096 - / - / 25 / 21
//   8 rows:  6000 columns 16 / 12 / 14 / -, 4096 of K = 4096 7.2 / 7.7 / 8.4 / -
//   32 rows: 16384 columns - / 43 / - / 32, 4096 of K = 4096 11 / 13 / - / 16
size_t matvecVariant(int64_t M, int64_t N) {
    const int64_t row_tiles = M <= 4 ? 0 : M <= 16 ? 1 : M <= 32 ? 2 : 4, tiles = (N + 15) / 16;
    size_t best = 0;
    int64_t least = INT64_MAX;
    for (size_t i = 0; i < std::size(kMatvecShapes); i++) {
        const MatvecShape &shape = kMatvecShapes[i];
        if (shape.row_tiles == row_tiles) {
            const int64_t workgroups = (tiles + shape.column_tiles - 1) / shape.column_tiles, rounds = (workgroups + 255) / 256;
            const int64_t work = rounds * (10 * shape.column_tiles + (row_tiles == 0 ? 7 : 20 * row_tiles));
            if (work < least) {
                least = work;
                best = i;
            }
        }
    }
    return best;
}

}  // namespace

int gern_matvec4_create(int64_t group, int type, int flags, gern_pipeline *out) {
    if (out == nullptr) {
        return fail("gern_matvec4_create: null argument");
    }
    *out = nullptr;
    if ((group != 32 && group != 64 && group != 128) || !goodType(type)) {
        return fail("gern_matvec4_create: group must be 32, 64 or 128, and type GERN_TYPE_BF16 or GERN_TYPE_F16");
    }
    try {
        Draft p(gern_pipeline_s::MATVEC4, flags);
        p->group = group;
        for (const MatvecShape &shape : kMatvecShapes) {
            AbstractDataTypePtr x(new const annot::WholeADT("x", "gernels::ActivationsOf<" + typeName(type) + ">"));
            AbstractDataTypePtr weights(new const annot::WholeADT("weights", "gernels::Weights4"));
            AbstractDataTypePtr y(new const annot::PiecesADT<hip::MatvecOut>("y", "gernels::MatvecOut", "at", {{"columns", &hip::MatvecOut::columns}}));
            annot::PieceFunction multiply("gernels::multiply_4bit", "gernels/serving/matvec4.h", {x, weights}, y, {"columns"},
                                          {"group", "row_tiles", "column_tiles", "waves"});
            Variable column("column"), threads("threads");
            Composable program =
                Global((Tile(y["columns"], column.bind(1)) || Grid::BLOCK_X)(
                           multiply[{constant("group", group), constant("row_tiles", shape.row_tiles), constant("column_tiles", shape.column_tiles),
                                     constant("waves", kMatvecWaves)}](x, weights, y)),
                       {{Grid::BLOCK_DIM_X, threads.bind(64 * kMatvecWaves)}});
            if (p.add(program, flags | GERN_PIPELINE_NO_XCD_REMAP) != 0) {
                return 1;
            }
        }
        *out = p.handOut();
    } catch (const std::exception &e) {
        return fail(e.what());
    }
    return 0;
}

int gern_matvec4_run(gern_pipeline p, const void *X, int64_t ldx, const uint8_t *codes, const void *scales, const uint8_t *zeros, void *Y, int64_t ldy,
                     int64_t M, int64_t N, int64_t K, void *stream) {
    if (!usable(p, gern_pipeline_s::MATVEC4)) {
        return fail("gern_matvec4_run: bad pipeline");
    }
    if (M < 0 || M > GERN_MATVEC4_MAX_ROWS || N < 1 || N > 0x7fffffff || K < 1 || K > GERN_MATVEC4_MAX_COLUMNS || K % p->group != 0) {
        return fail("gern_matvec4_run: M must be in [0, GERN_MATVEC4_MAX_ROWS = 64], N in [1, 2^31), K in [1, GERN_MATVEC4_MAX_COLUMNS = 2^24] and a "
                    "multiple of the group");
    }
    if (M == 0) {
        return 0;
    }
    if (X == nullptr || codes == nullptr || scales == nullptr || Y == nullptr) {
        return fail("gern_matvec4_run: null buffer");
    }
    if (!aligned(X, 16) || ldx % 8 != 0 || !aligned(codes, 16) || !aligned(scales, 2) || !aligned(Y, 2)) {
        return fail("gern_matvec4_run: X and the codes are read in 16-byte pieces: both must be 16-byte aligned and the row stride of X a multiple of 8 "
                    "elements (scales and Y 2-byte aligned)");
    }
    if (M > 1 && (ldx < K || ldx > 2 * GERN_MATVEC4_MAX_COLUMNS || ldy < N)) {
        return fail("gern_matvec4_run: a row stride is less than its row, or that of X more than 2 * GERN_MATVEC4_MAX_COLUMNS");
    }
    const int64_t x_bytes = ((M - 1) * ldx + K) * 2, y_bytes = ((M - 1) * ldy + N) * 2, groups = K / p->group;
    if (overlap(Y, y_bytes, X, x_bytes) || overlap(Y, y_bytes, codes, N * K / 2) || overlap(Y, y_bytes, scales, groups * N * 2) ||
        overlap(Y, y_bytes, zeros, zeros != nullptr ? groups * N : 0)) {
        return fail("gern_matvec4_run: Y shares memory with an input");
    }
    const size_t variant = matvecVariant(M, N);
    const int64_t tile = 16 * kMatvecShapes[variant].column_tiles;
    if (tooWide((N + tile - 1) / tile, 64 * kMatvecWaves)) {
        return fail("gern_matvec4_run: N must be less than 2^27");
    }
    hip::Activations x{X, ldx / 2, M};
    hip::Weights4 weights{codes, scales, zeros, N, K};
    hip::MatvecOut y{Y, ldy, (N + tile - 1) / tile};
    return evaluate(p, variant, "gern_matvec4_run", stream, {{"x", &x}, {"weights", &weights}, {"y", &y}});
}

}  // extern "C"
