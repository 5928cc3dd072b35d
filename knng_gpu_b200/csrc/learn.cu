// learn.cu -- C-ABI entry points of the projection and the softmax loss over
// inner products (include/knng_gpu.h) and their host-side orchestration.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <exception>
#include <mutex>
#include <string>

#include "internal.hpp"
#include "knng_gpu.h"
#include "learn.cuh"
#include "skinny.cuh"

using namespace knng_b200;

namespace {

knng_gpu_status fail(knng_gpu_status s, const std::string& msg) { return set_last_error(s, msg); }

#define KNNG_CUDA(call)                                                                          \
    do {                                                                                         \
        cudaError_t e_ = (call);                                                                 \
        if (e_ != cudaSuccess)                                                                   \
            return fail(e_ == cudaErrorMemoryAllocation ? KNNG_GPU_OUT_OF_MEMORY : KNNG_GPU_CUDA_ERROR, \
                        std::string("knng::gpu: ") + #call + ": " + cudaGetErrorString(e_));     \
    } while (0)

#define KNNG_TRY(expr)                        \
    do {                                      \
        knng_gpu_status s_ = (expr);          \
        if (s_ != KNNG_GPU_OK) return s_;     \
    } while (0)

constexpr uint64_t up(uint64_t x, uint64_t a) { return (x + a - 1) / a * a; }
constexpr uint64_t ceil_div(uint64_t x, uint64_t a) { return (x + a - 1) / a; }

uint32_t elem_bytes(int dtype) { return dtype == KNNG_DTYPE_F32 ? 4 : 2; }

// Number of bytes a call would need (base NULL), or the pieces of a workspace.
struct Carver {
    uint8_t* base;
    uint64_t at = 0;
    explicit Carver(void* b) : base(static_cast<uint8_t*>(b)) {}
    template <class T>
    T* take(uint64_t count)
    {
        T* p = base ? reinterpret_cast<T*>(base + at) : nullptr;
        at = up(at + count * sizeof(T), 256);
        return p;
    }
};

// ------------------------------------------------------------------ device facts
// Error word of the product kernel: host memory that kernels can write, so an
// asynchronous call needs no synchronisation to report a wait that gave up.
knng_gpu_status error_word(int** out)
{
    static std::mutex mu;
    static int* word = nullptr;
    std::lock_guard<std::mutex> lock(mu);
    if (!word) {
        void* p = nullptr;
        KNNG_CUDA(cudaHostAlloc(&p, sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped));
        word = static_cast<int*>(p);
        *word = 0;
    }
    *out = word;
    return KNNG_GPU_OK;
}

knng_gpu_status take_error(int** word)
{
    KNNG_TRY(error_word(word));
    if (reinterpret_cast<std::atomic<int>*>(*word)->exchange(0) != 0)
        return fail(KNNG_GPU_TIMEOUT, "knng::gpu: a bounded device wait gave up in an earlier call on device rows");
    return KNNG_GPU_OK;
}

uint32_t sm_count()
{
    static std::atomic<uint32_t> cached{0};
    uint32_t n = cached.load(std::memory_order_relaxed);
    if (n == 0) {
        int dev = 0, sms = 0;
        cudaGetDevice(&dev);
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
        n = sms > 0 ? static_cast<uint32_t>(sms) : 148u;
        if (sms > 0) cached.store(n, std::memory_order_relaxed);
    }
    return n;
}

// Launch in the stream's order, but allowed to be set up while the kernel
// before it drains: every kernel here waits for that one (previous_done) before
// it touches memory. A chain of short kernels saves 1 to 2 us per link.
template <class... P, class... A>
knng_gpu_status launch(void (*kern)(P...), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t st, A&&... args)
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    KNNG_CUDA(cudaLaunchKernelEx(&cfg, kern, P(args)...));
    return KNNG_GPU_OK;
}

// ------------------------------------------------------------------ maps
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

knng_gpu_status encode_fn(EncodeTiledFn* out)
{
    static std::atomic<void*> cached{nullptr};
    void* p = cached.load(std::memory_order_acquire);
    if (!p) {
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !p)
            return fail(KNNG_GPU_CUDA_ERROR, "knng::gpu: cuTensorMapEncodeTiled entry point not available");
        cached.store(p, std::memory_order_release);
    }
    *out = reinterpret_cast<EncodeTiledFn>(p);
    return KNNG_GPU_OK;
}

// rows x width elements at stride `ld`; boxes of box_w x box_h elements,
// swizzled over their width of 64 or 128 bytes; zeros past the ends.
knng_gpu_status make_map(CUtensorMap* map, int type, const void* base, uint64_t width, uint64_t rows, uint64_t ld,
                         uint32_t box_w, uint32_t box_h)
{
    if (!base) return fail(KNNG_GPU_INVALID_ARGUMENT, "knng::gpu: a matrix of a product is NULL");
    EncodeTiledFn enc;
    KNNG_TRY(encode_fn(&enc));
    const uint32_t e = elem_bytes(type);
    const CUtensorMapDataType dt = type == KNNG_DTYPE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : type == KNNG_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                             : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const cuuint64_t dims[2] = {width, rows};
    const cuuint64_t strides[1] = {ld * e};
    const cuuint32_t box[2] = {box_w, box_h};
    const cuuint32_t estr[2] = {1, 1};
    const CUtensorMapSwizzle sw = box_w * e == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    const CUresult r = enc(map, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           sw, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(KNNG_GPU_CUDA_ERROR, "knng::gpu: cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
    return KNNG_GPU_OK;
}

// TMA reads and writes rows that start on 16-byte boundaries.
bool tma_rows(const void* p, uint64_t ld, uint32_t e)
{
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * e) % 16 == 0;
}

// ------------------------------------------------------------------ operands
// A matrix that the product reads: `rows` stored rows of `width` 16-bit
// elements (all planes), `ld` apart.
struct Operand {
    const void* ptr;
    uint64_t rows, width, ld;
    uint32_t plane;  // columns from one plane to the next
};

struct Source {  // a caller's matrix
    const void* ptr;
    uint64_t rows, k, ld;
};

bool needs_stage(const Source& s, int dtype) { return dtype == KNNG_DTYPE_F32 || !tma_rows(s.ptr, s.ld, 2); }
uint32_t planes_of(int dtype) { return dtype == KNNG_DTYPE_F32 ? 3u : 1u; }
// Columns of a staged plane: 16-byte rows; whole K blocks where planes lie side by side.
uint64_t stage_pitch(uint64_t k, int dtype) { return dtype == KNNG_DTYPE_F32 ? up(k, 64) : up(k, 8); }

uint64_t stage_elems(const Source& s, int dtype) { return s.rows * stage_pitch(s.k, dtype) * planes_of(dtype); }

struct RowLabels {
    const void* ptr = nullptr;
    int i64 = 0;
    uint32_t classes = 0;
};

// The work of staging s at dst (none where dst is NULL).
StageJob stage_job(const Source& s, int dtype, uint16_t* dst, const RowLabels& labels = RowLabels())
{
    StageJob j = {};
    if (!dst) return j;
    j.x = s.ptr;
    j.rows = s.rows;
    j.k = static_cast<uint32_t>(s.k);
    j.ld = s.ld;
    j.out = dst;
    j.pitch = static_cast<uint32_t>(stage_pitch(s.k, dtype));
    j.labels = labels.ptr;
    j.labels_i64 = labels.i64;
    j.classes = labels.classes;
    j.blocks = static_cast<uint32_t>(std::min<uint64_t>(ceil_div(s.rows * (j.pitch / 8), 256), 148ull * 16));
    return j;
}

// The operand as the product reads it: staged at dst, or as the caller has it.
Operand operand(const Source& s, int dtype, const uint16_t* dst)
{
    if (!dst) return Operand{s.ptr, s.rows, s.k, s.ld, 0};
    const uint64_t pitch = stage_pitch(s.k, dtype), width = pitch * planes_of(dtype);
    return Operand{dst, s.rows, width, width, static_cast<uint32_t>(pitch)};
}

knng_gpu_status prepare(int dtype, const StageJob& a, const StageJob& b, const GradRowsJob& rows, cudaStream_t st)
{
    const uint32_t blocks = a.blocks + b.blocks + rows.blocks;
    if (blocks == 0) return KNNG_GPU_OK;
    return dtype == KNNG_DTYPE_F32 ? launch(prepare_kernel<3>, dim3(blocks), 256, 0, st, PrepareParams{a, b, rows})
                                   : launch(prepare_kernel<1>, dim3(blocks), 256, 0, st, PrepareParams{a, b, rows});
}

knng_gpu_status finish(const SumsJob& sums, const JoinParams& a, const JoinParams& b, cudaStream_t st)
{
    const uint32_t blocks = sums.blocks + a.blocks + b.blocks;
    if (blocks == 0) return KNNG_GPU_OK;
    return launch(finish_kernel, dim3(blocks), 256, 0, st, FinishParams{sums, a, b});
}

uint32_t join_blocks(uint64_t m, uint64_t n)
{
    return static_cast<uint32_t>(std::min<uint64_t>(ceil_div(m * ceil_div(n, 4), 256), 148ull * 16));
}

// ------------------------------------------------------------------ product launches
struct Shape {
    uint64_t m, n, k;
    uint32_t combos;
    bool precise;  // the result is kept in fp32
    bool bf16;     // operands are single bf16 values
};

// K blocks of 64 summed by the tensor cores alone, whose additions truncate:
// 1024 of K where 16 bits come of it, 256 (bf16) or 128 (fp16, whose products
// are longer) where the result stays fp32, 64 for six plane products. Loss of 2048 rows of
// width 960 against 30,000, relative error against 64 bits: bf16 1.3e-6 at 128,
// 2.4e-6 at 256 (and 1046 us instead of 1257 for 8192 rows against 100,000);
// fp16 2.3e-6 and 5.5e-6; plain fp32 3.6e-6 and 4.4e-6. A 16-bit result has
// 2e-4 or more of its own.
uint32_t piece_blocks(const Shape& s) { return !s.precise ? 16u : s.bf16 ? 4u : s.combos == 1 ? 2u : 1u; }

struct Plan {
    int cg;
    uint32_t tile_n, tiles_m, tiles_n, kblocks, splits, piece;
    uint32_t pieces() const { return (kblocks + piece - 1) / piece; }
    uint64_t split_rows, part_pitch;  // of the fp32 pieces of a split product
    uint64_t part_elems() const { return splits > 1 ? splits * split_rows * part_pitch : 0; }
};

Plan tiles_of(const Shape& s, int cg, uint32_t tile_n)
{
    Plan q;
    q.cg = cg;
    q.tile_n = tile_n;
    q.tiles_m = static_cast<uint32_t>(ceil_div(s.m, 128 * cg));
    q.tiles_n = static_cast<uint32_t>(ceil_div(s.n, tile_n));
    q.kblocks = static_cast<uint32_t>(ceil_div(s.k, 64));
    q.splits = 1;
    // As few pieces as the longest allows, all about as long.
    q.piece = static_cast<uint32_t>(ceil_div(q.kblocks, ceil_div(q.kblocks, piece_blocks(s))));
    q.split_rows = uint64_t(q.tiles_m) * 128 * cg;
    q.part_pitch = uint64_t(q.tiles_n) * tile_n;
    return q;
}

// Clock cycles of a product by its plan: rounds of items over the units, each
// item its K blocks and a fixed part (first loads, last stores, schedule); a
// launch of pairs takes some 3 us longer to get going than one of single CTAs.
// A K block costs the tensor cores 2 cycles per column of the tile (a pair
// does 256 rows at once, a single CTA 128) and plane product. Its 16 KiB of A
// and 128 bytes per row of B, for each plane, come from L2 at about 60 bytes a
// cycle and go into shared memory, from where every product reads its share at
// 128 bytes a cycle (six plane products: A and all of the tile's B each time, a
// pair's other half from its peer): single tiles and narrow ones are bound by
// that. A split product is written and read in fp32 once more, some 3400 bytes
// a cycle, and may need another kernel to join it.
double block_cycles(const Plan& q, const Shape& s)
{
    const double planes = s.combos == 1 ? 1.0 : 3.0;
    const double in = planes * (16384.0 + 128.0 * q.tile_n / q.cg);
    const double read = s.combos * (16384.0 + 128.0 * q.tile_n);
    const double l2 = in / 60.0;
    if (s.combos == 1) return std::max({2.0 * q.tile_n, 2.0 * in / 128.0, l2});
    return std::max({2.0 * s.combos * q.tile_n, (in + read) / 128.0, l2});
}

// Exponentials of a tile, 16 a cycle.
double exp_cycles(const Plan& q) { return 128.0 * q.tile_n / 16.0; }

double plan_cycles(const Plan& q, const Shape& s, bool exps = false)
{
    const uint64_t units = sm_count() / q.cg;
    const uint64_t items = uint64_t(q.tiles_m) * q.tiles_n * q.splits;
    const double rounds = static_cast<double>(ceil_div(items, units));
    double item = static_cast<double>(ceil_div(q.pieces(), q.splits)) * q.piece * block_cycles(q, s);
    if (exps) item = std::max(item, exp_cycles(q));
    double cycles = rounds * (item + 1500.0) + (q.cg == 2 ? 6000.0 : 0.0);
    if (q.splits > 1) cycles += 6000.0 + static_cast<double>(s.m) * s.n * q.splits * 8.0 / 3400.0;
    return cycles;
}

// The K loop cut into about `want` splits of equal length, each a whole number
// of pieces no longer than `whole`.
Plan cut_k(Plan q, uint32_t whole, uint64_t want)
{
    const uint64_t length = ceil_div(q.kblocks, want);
    const uint64_t per_split = ceil_div(length, whole);
    q.piece = static_cast<uint32_t>(ceil_div(length, per_split));
    q.splits = static_cast<uint32_t>(ceil_div(q.pieces(), per_split));
    return q;
}

// The cheapest of pairs (256 rows) and single CTAs (128 rows) with tiles from
// 64 columns up, the K loop whole or cut into 2, 3, 4, 6, 8, ... splits of at
// least four K blocks: where the tiles leave units idle, up to as many as fill
// them; where they do not, up to eight, to even out the last round.
Plan search_plan(const Shape& s, int only_cg)
{
    Plan best;
    double least = 0.0;
    for (int cg = 2; cg >= 1; --cg) {
        if (only_cg && cg != only_cg) continue;
        for (uint32_t tile_n = 128 * cg; tile_n >= 64u * cg; tile_n -= 32) {
            const Plan uncut = tiles_of(s, cg, tile_n);
            Plan q = uncut;
            const uint64_t tiles = uint64_t(q.tiles_m) * q.tiles_n;
            const uint64_t units = sm_count() / cg;
            const uint64_t longest = q.kblocks / ceil_div(4, s.combos);
            const uint64_t most = std::max<uint64_t>(
                1, std::min<uint64_t>(tiles < units ? units / tiles : tiles < 8 * units ? 8 : 1, longest));
            for (uint64_t want = 1;;) {
                q = cut_k(uncut, piece_blocks(s), want);
                const double c = plan_cycles(q, s);
                if (least == 0.0 || c < least) {
                    least = c;
                    best = q;
                }
                if (want == most) break;
                want = std::min(want < 4 ? want + 1 : want % 3 ? want + want / 2 : want + want / 3, most);
            }
        }
    }
    return best;
}

bool same(const Shape& a, const Shape& b)
{
    return a.m == b.m && a.n == b.n && a.k == b.k && a.combos == b.combos && a.precise == b.precise && a.bf16 == b.bf16;
}

uint64_t shape_key(const Shape& s)
{
    const uint64_t key = (s.m * 0x9E3779B97F4A7C15ull + s.n) * 0xC2B2AE3D27D4EB4Full + s.k * 0x165667B19E3779F9ull +
                         s.combos * 4 + s.precise * 2 + s.bf16;
    return key ^ (key >> 29);
}

// The search takes some microseconds of host time: a thread keeps the plans of
// the shapes it met last. `cg` 1 or 2 asks for that kind of tile, 0 for either.
Plan plan_product(const Shape& s, int cg = 0)
{
    struct Entry {
        Shape s;
        int cg;
        Plan q;
    };
    thread_local Entry kept[128] = {};
    Entry& e = kept[(shape_key(s) + cg) & 127];
    if (!same(e.s, s) || e.cg != cg) e = Entry{s, cg, search_plan(s, cg)};
    return e.q;
}

// The longest turn of a unit when the items of a, then those of b, are dealt
// out in a row.
double merged_cycles(const Plan& a, const Shape& sa, const Plan& b, const Shape& sb)
{
    const uint64_t units = sm_count() / a.cg;
    const uint64_t na = uint64_t(a.tiles_m) * a.tiles_n * a.splits, all = na + uint64_t(b.tiles_m) * b.tiles_n * b.splits;
    const double ca = static_cast<double>(ceil_div(a.pieces(), a.splits)) * a.piece * block_cycles(a, sa) + 1500.0;
    const double cb = static_cast<double>(ceil_div(b.pieces(), b.splits)) * b.piece * block_cycles(b, sb) + 1500.0;
    double longest = 0.0;
    for (const uint64_t u : {uint64_t(0), na % units, na % units + units - 1, all % units, all % units + units - 1}) {
        const uint64_t i = u % units;
        const uint64_t of_a = na / units + (i < na % units), of_all = all / units + (i < all % units);
        longest = std::max(longest, static_cast<double>(of_a) * ca + static_cast<double>(of_all - of_a) * cb);
    }
    if (a.splits > 1) longest += static_cast<double>(sa.m) * sa.n * a.splits * 8.0 / 3400.0;
    if (b.splits > 1) longest += static_cast<double>(sb.m) * sb.n * b.splits * 8.0 / 3400.0;
    return longest + (a.cg == 2 ? 6000.0 : 0.0);
}

struct TwoPlans {
    Plan a, b;
    bool merged;
};

// Plans of two products of one backward pass, and whether they run in one
// launch: that saves a launch and half-empty rounds where they are short
// (gradients of 1537 x 960 -> 300: 26.0 -> 23.2 us, of the loss of 4000 x 500
// against 8000: 141 -> 118 us). Not where they are long (100,000 x 784 -> 1024:
// 489 -> 505 us), and earlier not where only one of them sums a long K: the
// other would share its eight epilogue warps instead of having sixteen
// (100,000 x 784 -> 256: 129 -> 147 us, with odd rows of 785 242 -> 424). In one
// launch the splits are chosen so that the items of both fill the units
// together.
TwoPlans search_two(const Shape& a, const Shape& b)
{
    TwoPlans r{plan_product(a), plan_product(b), false};
    const bool alike = (r.a.pieces() > r.a.splits) == (r.b.pieces() > r.b.splits);
    if (plan_cycles(r.a, a) + plan_cycles(r.b, b) > (alike ? 2e5 : 6e4)) return r;
    r.merged = true;
    double least = 0.0;
    for (int cg = 2; cg >= 1; --cg) {
        const Plan qa = plan_product(a, cg), qb = plan_product(b, cg);
        const uint64_t units = sm_count() / cg;
        const auto most = [&](const Plan& q, const Shape& s) {
            const uint64_t tiles = uint64_t(q.tiles_m) * q.tiles_n;
            return std::max<uint64_t>(1, std::min<uint64_t>(tiles < units ? units / tiles : 1, q.kblocks / ceil_div(4, s.combos)));
        };
        const Plan ua = tiles_of(a, cg, qa.tile_n), ub = tiles_of(b, cg, qb.tile_n);
        for (uint64_t wa = 1; wa <= most(qa, a); ++wa)
            for (uint64_t wb = 1; wb <= most(qb, b); wb += wb < 4 ? 1 : wb / 2) {
                const Plan ca = cut_k(ua, piece_blocks(a), wa), cb = cut_k(ub, piece_blocks(b), wb);
                const double c = merged_cycles(ca, a, cb, b);
                if (least == 0.0 || c < least) {
                    least = c;
                    r.a = ca;
                    r.b = cb;
                }
            }
    }
    return r;
}

bool plan_two(const Shape& a, const Shape& b, Plan* qa, Plan* qb)
{
    struct Entry {
        Shape a, b;
        TwoPlans r;
    };
    thread_local Entry kept[64] = {};
    Entry& e = kept[(shape_key(a) * 31 + shape_key(b)) & 63];
    if (!same(e.a, a) || !same(e.b, b)) e = Entry{a, b, search_two(a, b)};
    *qa = e.r.a;
    *qb = e.r.b;
    return e.r.merged;
}

// Opts a kernel in to `bytes` of dynamic shared memory, once per device.
template <auto KERN>
knng_gpu_status allow_smem(uint32_t bytes)
{
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    KNNG_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (dev > 63 || !(done.load(std::memory_order_acquire) & bit)) {
        KNNG_CUDA(cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes)));
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
    return KNNG_GPU_OK;
}

template <int CG, int EPI, bool LONG, int N, int LAY>
knng_gpu_status launch_product_t(const ProductCall<N>& call, cudaStream_t st)
{
    constexpr auto* kern = product_kernel<CG, EPI, LONG, N, LAY>;
    // Units that fit the device at once (the same on every GPU this library is built for).
    static std::atomic<uint32_t> fit{0};
    uint32_t units = fit.load(std::memory_order_acquire);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CG;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.blockDim = dim3(pk_threads(CG, EPI, LONG));
    cfg.dynamicSmemBytes = kPkSmem;
    cfg.stream = st;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    KNNG_TRY(allow_smem<kern>(kPkSmem));
    if (units == 0) {
        // The kernel's roles trade registers within what the launch gives them.
        constexpr int kWarps = pk_epi_warps(CG, EPI, LONG);
        static_assert(4 * pk_issue_regs(kWarps) + kWarps * pk_epi_regs(kWarps) <= (4 + kWarps) * pk_launch_regs(kWarps),
                      "register split");
        cudaFuncAttributes fa;
        KNNG_CUDA(cudaFuncGetAttributes(&fa, kern));
        if (fa.numRegs < pk_launch_regs(kWarps))
            return fail(KNNG_GPU_CUDA_ERROR, "knng::gpu: product kernel built with too few registers");
        units = sm_count() / CG;
        if (CG == 2) {
            int clusters = 0;
            cfg.gridDim = dim3(sm_count() / 2 * 2);
            KNNG_CUDA(cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg));
            units = static_cast<uint32_t>(std::max(1, std::min<int>(clusters, static_cast<int>(units))));
        }
        fit.store(units, std::memory_order_release);
    }
    uint32_t items = call.p[0].items;
    if (N == 2) items += call.p[N - 1].items;
    cfg.gridDim = dim3(std::min(units, items) * CG);
    cfg.numAttrs = 2;
    KNNG_CUDA(cudaLaunchKernelEx(&cfg, kern, call));
    return KNNG_GPU_OK;
}

template <int EPI, int N, int LAY>
knng_gpu_status launch_product_l(int cg, const ProductCall<N>& call, cudaStream_t st)
{
    bool longk = call.p[0].pieces > call.p[0].splits;
    if (N == 2) longk = longk || call.p[N - 1].pieces > call.p[N - 1].splits;
    if (cg == 2)
        return longk ? launch_product_t<2, EPI, true, N, LAY>(call, st) : launch_product_t<2, EPI, false, N, LAY>(call, st);
    return longk ? launch_product_t<1, EPI, true, N, LAY>(call, st) : launch_product_t<1, EPI, false, N, LAY>(call, st);
}

template <int EPI, int N>
knng_gpu_status launch_product(int cg, const ProductCall<N>& call, cudaStream_t st)
{
    if constexpr (N == 2) {
        return launch_product_l<EPI, N, kAnyLayout>(cg, call, st);
    } else {
        if constexpr (EPI == kEpiStore) {
            if (call.p[0].layout == kKMN) return launch_product_l<EPI, N, kKMN>(cg, call, st);
            if (call.p[0].layout == kMNMN) return launch_product_l<EPI, N, kMNMN>(cg, call, st);
        }
        return launch_product_l<EPI, N, kKK>(cg, call, st);
    }
}

knng_gpu_status operand_maps(const Plan& q, const Operand& a, const Operand& b, Layout lay, int in_type, CUtensorMap* ma,
                             CUtensorMap* mb)
{
    KNNG_TRY(make_map(ma, in_type, a.ptr, a.width, a.rows, a.ld, 64, lay == kMNMN ? 64 : 128));
    return make_map(mb, in_type, b.ptr, b.width, b.rows, b.ld, 64, lay == kKK ? q.tile_n / q.cg : 64);
}

int operand_type(int dtype) { return dtype == KNNG_DTYPE_F16 ? kF16 : kBF16; }

ProductParams base_params(const Shape& s, const Plan& q, const Operand& a, const Operand& b, Layout lay, int dtype,
                          int* err)
{
    ProductParams p = {};
    p.m = static_cast<uint32_t>(s.m);
    p.n = static_cast<uint32_t>(s.n);
    p.tile_n = q.tile_n;
    p.tiles_m = q.tiles_m;
    p.tiles_n = q.tiles_n;
    p.splits = q.splits;
    p.segments = 1;
    p.items = q.tiles_m * q.tiles_n * q.splits;
    p.kblocks = q.kblocks;
    p.piece = q.piece;
    p.pieces = q.pieces();
    p.planes = s.combos == 1 ? 1 : 3;
    p.plane_a = a.plane;
    p.plane_b = b.plane;
    p.in_type = operand_type(dtype);
    p.layout = lay;
    p.error = err;
    p.wait_limit = kSpinLimitCycles;
    p.alpha = 1.0f;
    return p;
}

// What follows a product: the linear epilogue.
struct Tail {
    void* out;
    uint64_t ldo;
    int out_type;
    void* pre = nullptr;
    uint64_t ldp = 0;
    const void* bias = nullptr;
    const void* residual = nullptr;
    uint64_t ldr = 0;
    int aux_type = KNNG_DTYPE_BF16;
    int activation = KNNG_ACT_NONE;
    float alpha = 1.0f;
    const float* alpha_dev = nullptr;
    uint32_t alpha_parts = 0;
};

// Product i of a call: D = A B^T through the tail; where the plan splits K,
// the pieces go to `part` and the work of joining them into *join.
template <int N>
knng_gpu_status set_store(ProductCall<N>& call, int i, const Shape& s, const Plan& q, const Operand& a, const Operand& b,
                          Layout lay, int dtype, const Tail& t, float* part, JoinParams* join, int* err)
{
    KNNG_TRY(operand_maps(q, a, b, lay, operand_type(dtype), &call.map_a[i], &call.map_b[i]));
    ProductParams& p = call.p[i];
    p = base_params(s, q, a, b, lay, dtype, err);
    call.map_out[i] = call.map_a[i];
    call.map_pre[i] = call.map_a[i];
    if (q.splits > 1) {
        p.out = part;
        p.out_type = kF32;
        p.out_tma = 1;
        p.split_rows = static_cast<uint32_t>(q.split_rows);
        JoinParams& j = *join;
        j.part = part;
        j.splits = q.splits;
        j.split_rows = q.split_rows;
        j.pitch = static_cast<uint32_t>(q.part_pitch);
        j.m = s.m;
        j.n = static_cast<uint32_t>(s.n);
        j.alpha = t.alpha;
        j.alpha_dev = t.alpha_dev;
        j.alpha_parts = t.alpha_parts;
        j.bias = t.bias;
        j.residual = t.residual;
        j.ldr = t.ldr;
        j.aux_type = t.aux_type;
        j.activation = t.activation;
        j.out = t.out;
        j.ldo = t.ldo;
        j.out_type = t.out_type;
        j.pre = t.pre;
        j.ldp = t.ldp;
        j.blocks = join_blocks(s.m, s.n);
        return make_map(&call.map_out[i], KNNG_DTYPE_F32, part, q.part_pitch, q.splits * q.split_rows, q.part_pitch, 32, 32);
    }
    p.out = t.out;
    p.ldo = t.ldo;
    p.out_type = t.out_type;
    p.out_tma = tma_rows(t.out, t.ldo, elem_bytes(t.out_type));
    p.pre = t.pre;
    p.ldp = t.ldp;
    p.pre_tma = t.pre && tma_rows(t.pre, t.ldp, elem_bytes(t.aux_type));
    p.bias = t.bias;
    p.bias_vec = (reinterpret_cast<uintptr_t>(t.bias) & 15) == 0;
    p.residual = t.residual;
    p.ldr = t.ldr;
    p.aux_type = t.aux_type;
    p.residual_vec = t.residual && tma_rows(t.residual, t.ldr, elem_bytes(t.aux_type));
    p.activation = t.activation;
    p.alpha = t.alpha;
    p.alpha_dev = t.alpha_dev;
    p.alpha_parts = t.alpha_parts;
    if (p.out_tma) KNNG_TRY(make_map(&call.map_out[i], t.out_type, t.out, s.n, s.m, t.ldo, 32, 32));
    if (p.pre_tma) KNNG_TRY(make_map(&call.map_pre[i], t.aux_type, t.pre, s.n, s.m, t.ldp, 32, 32));
    return KNNG_GPU_OK;
}

// ------------------------------------------------------------------ checks
constexpr uint64_t kMaxRows = (1ull << 31) - 512;
constexpr uint64_t kMaxWidth = 1ull << 20;

knng_gpu_status check_matrix(const char* op, const char* name, const void* p, uint64_t rows, uint64_t width,
                             uint64_t ld, int dtype)
{
    if (rows && !p) return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": " + name + " is NULL");
    if (ld < width)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": row stride of " + name + " (" + std::to_string(ld) +
                                                   ") must be >= its width (" + std::to_string(width) + ")");
    if (reinterpret_cast<uintptr_t>(p) % elem_bytes(dtype))
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": " + name + " is not aligned to its elements");
    return KNNG_GPU_OK;
}

knng_gpu_status check_sizes(const char* op, uint64_t m, uint64_t k, uint64_t n, int dtype)
{
    if (dtype != KNNG_DTYPE_F32 && dtype != KNNG_DTYPE_BF16 && dtype != KNNG_DTYPE_F16)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": unknown dtype " + std::to_string(dtype));
    if (k == 0) return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": k must be > 0");
    if (n == 0) return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": n must be > 0");
    if (m > kMaxRows || n > kMaxRows || k > kMaxWidth)
        return fail(KNNG_GPU_NOT_SUPPORTED, std::string(op) + ": m and n must be < 2^31 - 512, k <= 2^20");
    return KNNG_GPU_OK;
}

// Work items are counted in 32 bits.
knng_gpu_status check_items(const char* op, const Plan& q)
{
    if (uint64_t(q.tiles_m) * q.tiles_n * q.splits >= (1ull << 31))
        return fail(KNNG_GPU_NOT_SUPPORTED, std::string(op) + ": too many output tiles in one call");
    return KNNG_GPU_OK;
}

knng_gpu_status check_workspace(const char* op, const void* ws, uint64_t have, uint64_t need)
{
    if (need == 0) return KNNG_GPU_OK;
    if (!ws || have < need)
        return fail(KNNG_GPU_WORKSPACE_TOO_SMALL, std::string(op) + ": workspace of " + std::to_string(have) +
                                                      " bytes, needs " + std::to_string(need));
    if (reinterpret_cast<uintptr_t>(ws) & 255)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": workspace must be 256-byte aligned");
    return KNNG_GPU_OK;
}

// ------------------------------------------------------------------ few rows
// Few rows of x go to the skinny kernel, its shared memory permitting. Against
// the product kernel (padded to 128 rows), a linear layer of 16 bf16 rows takes
// 6.3 us instead of 7.2 at 960 -> 1024 and the same 45 us at 960 -> 100,000,
// one of 8 rows 4.4 and 38 us. Operands that would have to be staged first go
// there, sixteen rows to a block, while that is cheaper than the launch and the
// copy: up to 64 rows while w is small enough to be read several times from L2
// (fp16 33 x 785 -> 300: 8.0 us instead of 10.9), and up to 2^24 products (bf16
// 2000 x 61 -> 100: 4.9 us instead of 6.2, but 15.4 instead of 9.5 at 4e7), of
// fp32 rows for 256 of them (100 x 300 -> 300: 7.3 us instead of 11.0). The 256
// is no crossing point: 1000 x 100 -> 100 would take 6.4 us instead of 8.6, and
// only near 2e7 products is it slower (5000 x 64 -> 64: 10.4 instead of 7.4). It
// keeps the product kernel, and a workspace, for fp32 calls of a few hundred rows.
bool is_skinny(const Source& x, const Source& w, int dtype)
{
    if (x.k > kMaxWidth / 2 || up(std::min<uint64_t>(x.rows, kSkinnyRows), 8) *
                                       skinny_pitch(static_cast<uint32_t>(x.k), dtype == KNNG_DTYPE_F32) > kSkinnySmem)
        return false;
    if (x.rows <= kSkinnyRows) return true;
    if (x.rows > kSkinnyRows * 65535ull || !(needs_stage(x, dtype) || needs_stage(w, dtype))) return false;
    if (x.rows <= 4 * kSkinnyRows && w.rows * w.k <= (2ull << 20)) return true;
    return (dtype != KNNG_DTYPE_F32 || x.rows <= 256) &&
           static_cast<double>(x.rows) * static_cast<double>(w.rows) * static_cast<double>(x.k) <= 16777216.0;
}

struct SkinnyPlan {
    uint32_t ksplit, blocks;
};

// Warps: at least eight per SM by cutting K where w has few rows; at most four
// blocks of eight warps per SM, which then walk over w.
SkinnyPlan plan_skinny(uint64_t n, uint64_t k, int dtype)
{
    const uint64_t groups = ceil_div(n, 16), steps = ceil_div(k, skinny_step(dtype == KNNG_DTYPE_F32));
    SkinnyPlan q{1, 1};
    while (q.ksplit < 8 && groups * q.ksplit < sm_count() * 8ull && steps >= 2 * q.ksplit) q.ksplit *= 2;
    q.blocks = static_cast<uint32_t>(std::min<uint64_t>(ceil_div(groups, 8 / q.ksplit), sm_count() * 4ull));
    return q;
}

template <int TYPE, int NT, int EPI>
knng_gpu_status launch_skinny_t(const SkinnyParams& p, uint32_t blocks, cudaStream_t st)
{
    constexpr auto* kern = skinny_kernel<TYPE, NT, EPI>;
    const uint32_t smem = NT * 8 * p.pitch;
    if (smem > 16 * 1024) KNNG_TRY(allow_smem<kern>(kSkinnySmem));
    return launch(kern, dim3(blocks, (p.m + kSkinnyRows - 1) / kSkinnyRows), 256, smem, st, p);
}

template <int TYPE, int EPI>
knng_gpu_status launch_skinny_n(const SkinnyParams& p, uint32_t blocks, cudaStream_t st)
{
    return p.m <= 8 ? launch_skinny_t<TYPE, 1, EPI>(p, blocks, st) : launch_skinny_t<TYPE, 2, EPI>(p, blocks, st);
}

template <int EPI>
knng_gpu_status launch_skinny(const SkinnyParams& p, int dtype, uint32_t blocks, cudaStream_t st)
{
    if (dtype == KNNG_DTYPE_BF16) return launch_skinny_n<kBF16, EPI>(p, blocks, st);
    if (dtype == KNNG_DTYPE_F16) return launch_skinny_n<kF16, EPI>(p, blocks, st);
    return launch_skinny_n<kF32, EPI>(p, blocks, st);
}

SkinnyParams skinny_params(const Source& x, const Source& w, int dtype, const SkinnyPlan& q)
{
    SkinnyParams p = {};
    p.x = x.ptr;
    p.ldx = x.ld;
    p.w = w.ptr;
    p.ldw = w.ld;
    p.m = static_cast<uint32_t>(x.rows);
    p.n = static_cast<uint32_t>(w.rows);
    p.k = static_cast<uint32_t>(x.k);
    p.pitch = skinny_pitch(p.k, dtype == KNNG_DTYPE_F32);
    p.ksplit = q.ksplit;
    p.x_vec = tma_rows(x.ptr, x.ld, elem_bytes(dtype));
    const uint32_t e = elem_bytes(dtype);
    p.w_vec = !tma_rows(w.ptr, w.ld, e) ? 0 : (reinterpret_cast<uintptr_t>(w.ptr) | w.ld * e) % 32 == 0 ? 2 : 1;
    return p;
}

// ------------------------------------------------------------------ linear
// With `need` the bytes of workspace only.
knng_gpu_status linear_run(const knng_gpu_linear_args& a, void* ws, uint64_t ws_bytes, cudaStream_t st, uint64_t* need)
{
    static const char* const op = "knng::gpu::linear";
    KNNG_TRY(check_sizes(op, a.m, a.k, a.n, a.dtype));
    if (a.out_dtype != a.dtype && a.out_dtype != KNNG_DTYPE_F32)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": out_dtype must be dtype or fp32");
    if (a.activation < KNNG_ACT_NONE || a.activation > KNNG_ACT_SILU)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": unknown activation " + std::to_string(a.activation));
    if (need) *need = 0;
    if (a.m == 0) return KNNG_GPU_OK;
    const Source x{a.x, a.m, a.k, a.ldx}, w{a.w, a.n, a.k, a.ldw};
    const Shape s{a.m, a.n, a.k, a.dtype == KNNG_DTYPE_F32 ? 6u : 1u, a.out_dtype == KNNG_DTYPE_F32,
                  a.dtype == KNNG_DTYPE_BF16};
    const bool skinny = is_skinny(x, w, a.dtype);
    const Plan q = skinny ? Plan{} : plan_product(s);
    if (skinny && need) return KNNG_GPU_OK;
    KNNG_TRY(check_items(op, q));
    Carver c(ws);
    uint16_t* xs = !skinny && needs_stage(x, a.dtype) ? c.take<uint16_t>(stage_elems(x, a.dtype)) : nullptr;
    uint16_t* wst = !skinny && needs_stage(w, a.dtype) ? c.take<uint16_t>(stage_elems(w, a.dtype)) : nullptr;
    float* part = q.splits > 1 ? c.take<float>(q.part_elems()) : nullptr;
    if (need) {
        *need = c.at;
        return KNNG_GPU_OK;
    }
    KNNG_TRY(check_matrix(op, "x", a.x, a.m, a.k, a.ldx, a.dtype));
    KNNG_TRY(check_matrix(op, "w", a.w, a.n, a.k, a.ldw, a.dtype));
    KNNG_TRY(check_matrix(op, "out", a.out, a.m, a.n, a.ldo, a.out_dtype));
    if (a.residual) KNNG_TRY(check_matrix(op, "residual", a.residual, a.m, a.n, a.ldr, a.dtype));
    if (a.pre) KNNG_TRY(check_matrix(op, "pre", a.pre, a.m, a.n, a.ldp, a.dtype));
    if (a.bias) KNNG_TRY(check_matrix(op, "bias", a.bias, 1, a.n, a.n, a.dtype));
    KNNG_TRY(check_workspace(op, ws, ws_bytes, c.at));
    if (skinny) {
        const SkinnyPlan sq = plan_skinny(a.n, a.k, a.dtype);
        SkinnyParams p = skinny_params(x, w, a.dtype, sq);
        p.bias = a.bias;
        p.residual = a.residual;
        p.ldr = a.ldr;
        p.out = a.out;
        p.ldo = a.ldo;
        p.out_type = a.out_dtype;
        p.pre = a.pre;
        p.ldp = a.ldp;
        p.activation = a.activation;
        return launch_skinny<kEpiStore>(p, a.dtype, sq.blocks, st);
    }
    int* err;
    KNNG_TRY(take_error(&err));
    KNNG_TRY(prepare(a.dtype, stage_job(x, a.dtype, xs), stage_job(w, a.dtype, wst), GradRowsJob{}, st));
    Tail t{a.out, a.ldo, a.out_dtype};
    t.pre = a.pre;
    t.ldp = a.ldp;
    t.bias = a.bias;
    t.residual = a.residual;
    t.ldr = a.ldr;
    t.aux_type = a.dtype;
    t.activation = a.activation;
    JoinParams join = {};
    ProductCall<1> call;
    KNNG_TRY(set_store(call, 0, s, q, operand(x, a.dtype, xs), operand(w, a.dtype, wst), kKK, a.dtype, t, part, &join, err));
    KNNG_TRY(launch_product<kEpiStore>(q.cg, call, st));
    return finish(SumsJob{}, join, JoinParams{}, st);
}

// ------------------------------------------------------------------ linear backward
template <int ACT>
knng_gpu_status launch_slope_t(const SlopeParams& p, int dtype, dim3 grid, cudaStream_t st)
{
    if (dtype == KNNG_DTYPE_BF16) return launch(slope_kernel<ACT, kBF16>, grid, 256, 0, st, p);
    if (dtype == KNNG_DTYPE_F16) return launch(slope_kernel<ACT, kF16>, grid, 256, 0, st, p);
    return launch(slope_kernel<ACT, kF32>, grid, 256, 0, st, p);
}

knng_gpu_status launch_slope(const SlopeParams& p, int activation, int dtype, dim3 grid, cudaStream_t st)
{
    switch (activation) {
        case KNNG_ACT_RELU: return launch_slope_t<kActRelu>(p, dtype, grid, st);
        case KNNG_ACT_GELU: return launch_slope_t<kActGelu>(p, dtype, grid, st);
        case KNNG_ACT_GELU_TANH: return launch_slope_t<kActGeluTanh>(p, dtype, grid, st);
        case KNNG_ACT_SILU: return launch_slope_t<kActSilu>(p, dtype, grid, st);
        default: return launch_slope_t<kActNone>(p, dtype, grid, st);
    }
}

knng_gpu_status linear_backward_run(const knng_gpu_linear_backward_args& a, void* ws, uint64_t ws_bytes,
                                    cudaStream_t st, uint64_t* need)
{
    static const char* const op = "knng::gpu::linear_backward";
    KNNG_TRY(check_sizes(op, a.m, a.k, a.n, a.dtype));
    if (a.activation < KNNG_ACT_NONE || a.activation > KNNG_ACT_SILU)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": unknown activation " + std::to_string(a.activation));
    if (need) *need = 0;
    const uint32_t e = elem_bytes(a.dtype);
    if (a.m == 0) {
        if (need) return KNNG_GPU_OK;
        if (a.dw) KNNG_CUDA(cudaMemsetAsync(a.dw, 0, a.n * a.k * e, st));
        if (a.db) KNNG_CUDA(cudaMemsetAsync(a.db, 0, a.n * e, st));
        return KNNG_GPU_OK;
    }
    if (a.activation != KNNG_ACT_NONE && !a.pre)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": pre is NULL with an activation");
    const bool f32 = a.dtype == KNNG_DTYPE_F32;
    const uint32_t combos = f32 ? 6 : 1;
    const Source dy{a.dy, a.m, a.n, a.lddy}, x{a.x, a.m, a.k, a.ldx}, w{a.w, a.n, a.k, a.ldw};
    const bool slope = a.activation != KNNG_ACT_NONE;
    const bool products = a.dx || a.dw;
    // dz lies in the workspace unless it is dy and TMA can read that.
    const bool make_dz = products && (slope || needs_stage(dy, a.dtype));
    const Shape sx{a.m, a.k, a.n, combos, f32, a.dtype == KNNG_DTYPE_BF16}, sw{a.n, a.k, a.m, combos, f32, a.dtype == KNNG_DTYPE_BF16};
    Plan qx = plan_product(sx), qw = plan_product(sw);
    const bool merged = a.dx && a.dw && plan_two(sx, sw, &qx, &qw);
    KNNG_TRY(check_items(op, qx));
    KNNG_TRY(check_items(op, qw));
    const uint64_t pitch = stage_pitch(a.n, a.dtype);
    const uint32_t gx = static_cast<uint32_t>(ceil_div(pitch, 256));
    const uint32_t gy = static_cast<uint32_t>(std::max<uint64_t>(
        1, std::min<uint64_t>(sm_count() * uint64_t(kSlopeBlocks) / gx, ceil_div(a.m, 8))));
    Carver c(ws);
    uint16_t* dz = make_dz ? c.take<uint16_t>(a.m * pitch * planes_of(a.dtype)) : nullptr;
    uint16_t* xs = a.dw && needs_stage(x, a.dtype) ? c.take<uint16_t>(stage_elems(x, a.dtype)) : nullptr;
    uint16_t* wst = a.dx && needs_stage(w, a.dtype) ? c.take<uint16_t>(stage_elems(w, a.dtype)) : nullptr;
    float* sums = a.db ? c.take<float>(uint64_t(gy) * a.n) : nullptr;
    float* xpart = a.dx && qx.splits > 1 ? c.take<float>(qx.part_elems()) : nullptr;
    float* wpart = a.dw && qw.splits > 1 ? c.take<float>(qw.part_elems()) : nullptr;
    if (need) {
        *need = c.at;
        return KNNG_GPU_OK;
    }
    KNNG_TRY(check_matrix(op, "dy", a.dy, a.m, a.n, a.lddy, a.dtype));
    if (a.dw) KNNG_TRY(check_matrix(op, "x", a.x, a.m, a.k, a.ldx, a.dtype));
    if (a.dx) KNNG_TRY(check_matrix(op, "w", a.w, a.n, a.k, a.ldw, a.dtype));
    if (slope) KNNG_TRY(check_matrix(op, "pre", a.pre, a.m, a.n, a.ldp, a.dtype));
    if (a.dx) KNNG_TRY(check_matrix(op, "dx", a.dx, a.m, a.k, a.k, a.dtype));
    if (a.dw) KNNG_TRY(check_matrix(op, "dw", a.dw, a.n, a.k, a.k, a.dtype));
    if (a.db) KNNG_TRY(check_matrix(op, "db", a.db, 1, a.n, a.n, a.dtype));
    KNNG_TRY(check_workspace(op, ws, ws_bytes, c.at));
    int* err;
    KNNG_TRY(take_error(&err));
    const StageJob stage_x = stage_job(x, a.dtype, xs), stage_w = stage_job(w, a.dtype, wst);
    SumsJob db = {};
    if (make_dz || a.db) {
        SlopeParams p = {};
        p.dy = a.dy;
        p.lddy = a.lddy;
        p.pre = slope ? a.pre : nullptr;
        p.ldp = a.ldp;
        p.m = a.m;
        p.n = static_cast<uint32_t>(a.n);
        p.out = dz;
        p.pitch = static_cast<uint32_t>(pitch);
        p.sums = sums;
        p.vec = tma_rows(a.dy, a.lddy, e) && (!slope || tma_rows(a.pre, a.ldp, e));
        p.gx = gx;
        p.gy = gy;
        p.a = stage_x;
        p.b = stage_w;
        KNNG_TRY(launch_slope(p, a.activation, a.dtype, dim3(gx * gy + stage_x.blocks + stage_w.blocks), st));
        if (a.db) db = SumsJob{sums, gy, static_cast<uint32_t>(a.n), a.db, a.dtype, static_cast<uint32_t>(ceil_div(a.n, 32))};
    } else {
        KNNG_TRY(prepare(a.dtype, stage_x, stage_w, GradRowsJob{}, st));
    }
    const Operand oz = make_dz ? Operand{dz, a.m, pitch * planes_of(a.dtype), pitch * planes_of(a.dtype),
                                         static_cast<uint32_t>(pitch)}
                               : operand(dy, a.dtype, nullptr);
    JoinParams join_x = {}, join_w = {};
    const Operand ow = operand(w, a.dtype, wst), ox = operand(x, a.dtype, xs);
    const Tail tx{a.dx, a.k, a.dtype}, tw{a.dw, a.k, a.dtype};
    if (merged) {
        ProductCall<2> call;
        KNNG_TRY(set_store(call, 0, sx, qx, oz, ow, kKMN, a.dtype, tx, xpart, &join_x, err));
        KNNG_TRY(set_store(call, 1, sw, qw, oz, ox, kMNMN, a.dtype, tw, wpart, &join_w, err));
        KNNG_TRY(launch_product<kEpiStore>(qx.cg, call, st));
    } else {
        ProductCall<1> call;
        if (a.dx) {
            KNNG_TRY(set_store(call, 0, sx, qx, oz, ow, kKMN, a.dtype, tx, xpart, &join_x, err));
            KNNG_TRY(launch_product<kEpiStore>(qx.cg, call, st));
        }
        if (a.dw) {
            KNNG_TRY(set_store(call, 0, sw, qw, oz, ox, kMNMN, a.dtype, tw, wpart, &join_w, err));
            KNNG_TRY(launch_product<kEpiStore>(qw.cg, call, st));
        }
    }
    return finish(db, join_x, join_w, st);
}

// ------------------------------------------------------------------ softmax loss
knng_gpu_status check_scale(const char* op, float scale)
{
    if (!(scale > 0.0f) || !std::isfinite(scale))
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": scale must be finite and > 0");
    return KNNG_GPU_OK;
}

// Pairs or single CTAs, and pieces of the columns per row tile: such that the
// (row tile, piece) items fill one to eight rounds of the units best, counting
// that the longest piece of a round sets its time.
struct SoftmaxPlan {
    Plan q;
    uint32_t segments;
};

SoftmaxPlan plan_softmax(const Shape& s)
{
    SoftmaxPlan best{};
    double least = 0.0;
    for (int cg = 2; cg >= 1; --cg) {
        const Plan q = tiles_of(s, cg, 128 * cg);
        const uint64_t units = sm_count() / cg;
        const double tile = std::max(q.kblocks * block_cycles(q, s), exp_cycles(q)) + 300.0;
        for (uint64_t rounds = 1; rounds <= 8; ++rounds) {
            const uint32_t seg = static_cast<uint32_t>(
                std::max<uint64_t>(1, std::min<uint64_t>(q.tiles_n, rounds * units / q.tiles_m)));
            const double longest = static_cast<double>(ceil_div(q.tiles_n, seg));
            const double turns = static_cast<double>(ceil_div(uint64_t(seg) * q.tiles_m, units));
            const double time = turns * (longest * tile + 1500.0) + (cg == 2 ? 6000.0 : 0.0);
            if (least == 0.0 || time < least) {
                least = time;
                best = SoftmaxPlan{q, seg};
            }
        }
    }
    return best;
}

knng_gpu_status softmax_xent_run(const knng_gpu_softmax_xent_args& a, void* ws, uint64_t ws_bytes, cudaStream_t st,
                                 uint64_t* need)
{
    static const char* const op = "knng::gpu::softmax_xent";
    KNNG_TRY(check_sizes(op, a.m, a.k, a.n, a.dtype));
    KNNG_TRY(check_scale(op, a.scale));
    if (need) *need = 0;
    if (a.m == 0) return KNNG_GPU_OK;
    const Source x{a.x, a.m, a.k, a.ldx}, w{a.w, a.n, a.k, a.ldw};
    const Shape s{a.m, a.n, a.k, a.dtype == KNNG_DTYPE_F32 ? 6u : 1u, true, a.dtype == KNNG_DTYPE_BF16};
    // Pairs unless they would leave SMs idle; then the columns are cut so that
    // (row tile, piece) items fill the units in whole rounds.
    const bool skinny = is_skinny(x, w, a.dtype);
    const SkinnyPlan sq = plan_skinny(a.n, a.k, a.dtype);
    const SoftmaxPlan plan = skinny ? SoftmaxPlan{} : plan_softmax(s);
    const Plan& q = plan.q;
    const uint32_t segments = plan.segments;
    KNNG_TRY(check_items(op, q));
    const uint32_t pieces =
        skinny ? sq.blocks : segments * (pk_epi_warps(q.cg, kEpiSoftmax, q.pieces() > 1) / 4);
    Carver c(ws);
    uint16_t* xs = !skinny && needs_stage(x, a.dtype) ? c.take<uint16_t>(stage_elems(x, a.dtype)) : nullptr;
    uint16_t* wst = !skinny && needs_stage(w, a.dtype) ? c.take<uint16_t>(stage_elems(w, a.dtype)) : nullptr;
    float2* part = c.take<float2>(uint64_t(pieces) * a.m);
    float* label_dot = c.take<float>(a.m);
    if (need) {
        *need = c.at;
        return KNNG_GPU_OK;
    }
    KNNG_TRY(check_matrix(op, "x", a.x, a.m, a.k, a.ldx, a.dtype));
    KNNG_TRY(check_matrix(op, "w", a.w, a.n, a.k, a.ldw, a.dtype));
    if (!a.labels || !a.loss || !a.lse) return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": labels, loss or lse is NULL");
    KNNG_TRY(check_workspace(op, ws, ws_bytes, c.at));
    const float scale2 = a.scale * 1.44269504088896f;
    if (skinny) {
        SkinnyParams p = skinny_params(x, w, a.dtype, sq);
        p.scale2 = scale2;
        p.labels = a.labels;
        p.labels_i64 = a.labels_i64;
        p.part = part;
        p.label_dot = label_dot;
        KNNG_TRY(launch_skinny<kEpiSoftmax>(p, a.dtype, sq.blocks, st));
    } else {
        int* err;
        KNNG_TRY(take_error(&err));
        KNNG_TRY(prepare(a.dtype, stage_job(x, a.dtype, xs), stage_job(w, a.dtype, wst), GradRowsJob{}, st));
        const Operand ox = operand(x, a.dtype, xs), ow = operand(w, a.dtype, wst);
        ProductCall<1> call;
        KNNG_TRY(operand_maps(q, ox, ow, kKK, operand_type(a.dtype), &call.map_a[0], &call.map_b[0]));
        call.map_out[0] = call.map_pre[0] = call.map_a[0];
        ProductParams& p = call.p[0];
        p = base_params(s, q, ox, ow, kKK, a.dtype, err);
        p.segments = segments;
        p.items = q.tiles_m * segments;
        p.scale2 = scale2;
        p.labels = a.labels;
        p.labels_i64 = a.labels_i64;
        p.classes = static_cast<uint32_t>(a.n);
        p.part = part;
        p.label_dot = label_dot;
        KNNG_TRY(launch_product<kEpiSoftmax>(q.cg, call, st));
    }
    // A block per row where there are few rows with many pieces, a warp per row otherwise.
    if (pieces > 64 && a.m < sm_count() * 8)
        return launch(join_softmax_kernel<256>, dim3(static_cast<uint32_t>(a.m)), 256, 0, st, part, pieces, a.m,
                      label_dot, scale2, a.labels, a.labels_i64, a.n, a.loss, a.lse);
    return launch(join_softmax_kernel<32>, dim3(static_cast<uint32_t>(ceil_div(a.m, 8))), 256, 0, st, part, pieces, a.m,
                  label_dot, scale2, a.labels, a.labels_i64, a.n, a.loss, a.lse);
}

// ------------------------------------------------------------------ softmax loss, gradient
// Most bytes of a piece's g: enough columns that the products of a piece fill
// the GPU for many rounds of tiles; a small part of all scores of a large call.
constexpr uint64_t kPieceBytes = 256ull << 20;

struct GradPlan {
    uint64_t width;      // columns of a piece, the last one narrower
    Plan g, dx, dw, dw_last;
    bool merged;         // dx and dw in one launch
};

Plan plan_grad_tiles(const Shape& s)
{
    Plan best{};
    double least = 0.0;
    for (int cg = 2; cg >= 1; --cg)
        for (uint32_t tile_n = 128 * cg; tile_n >= 64; tile_n -= 64 * cg) {  // 256 and 128, 128 and 64
            const Plan q = tiles_of(s, cg, tile_n);
            const double c = plan_cycles(q, s, true);
            if (least == 0.0 || c < least) {
                least = c;
                best = q;
            }
        }
    return best;
}

// Pieces: as few as their bytes allow, or a few more where that evens out the
// rounds of the three products (looked for only in calls of 0.2 ms and more).
GradPlan plan_grad(uint64_t m, uint64_t k, uint64_t n, int dtype)
{
    const uint32_t planes = planes_of(dtype), combos = planes == 3 ? 6 : 1;
    const bool f32 = planes == 3, bf16 = dtype == KNNG_DTYPE_BF16;
    const uint64_t widest = std::max<uint64_t>(2048, kPieceBytes / (2 * planes * m) / 256 * 256);
    const uint64_t fewest = ceil_div(n, widest);
    GradPlan best{};
    double least = 0.0;
    for (uint64_t pieces = fewest; pieces < fewest + 6; ++pieces) {
        GradPlan p;
        p.width = std::min(up(ceil_div(n, pieces), 256), n);
        if (pieces > fewest && p.width < 2048) break;
        const uint64_t count = ceil_div(n, p.width);
        const Shape sg{m, p.width, k, combos, f32, bf16}, sx{m, k, p.width, combos, f32, bf16};
        const Shape sw{p.width, k, m, combos, f32, bf16}, sl{n - (count - 1) * p.width, k, m, combos, f32, bf16};
        p.g = plan_grad_tiles(sg);
        p.merged = plan_two(sx, sw, &p.dx, &p.dw);
        p.dw_last = count > 1 ? plan_product(sl, p.merged ? p.dx.cg : 0) : p.dw;
        const double c = static_cast<double>(count) * (plan_cycles(p.g, sg, true) + plan_cycles(p.dx, sx) + plan_cycles(p.dw, sw));
        if (least == 0.0 || c < least) {
            least = c;
            best = p;
        }
        if (least < 4e5) break;
    }
    return best;
}

knng_gpu_status softmax_xent_backward_run(const knng_gpu_softmax_xent_backward_args& a, void* ws, uint64_t ws_bytes,
                                          cudaStream_t st, uint64_t* need)
{
    static const char* const op = "knng::gpu::softmax_xent_backward";
    KNNG_TRY(check_sizes(op, a.m, a.k, a.n, a.dtype));
    KNNG_TRY(check_scale(op, a.scale));
    if (need) *need = 0;
    const uint32_t e = elem_bytes(a.dtype);
    if (a.m == 0) {
        if (need || !a.dw) return KNNG_GPU_OK;
        KNNG_CUDA(cudaMemsetAsync(a.dw, 0, a.n * a.k * e, st));
        return KNNG_GPU_OK;
    }
    const uint32_t planes = planes_of(a.dtype);
    const uint32_t combos = planes == 3 ? 6 : 1;
    const Source x{a.x, a.m, a.k, a.ldx}, w{a.w, a.n, a.k, a.ldw};
    const bool f32 = planes == 3;
    const GradPlan plan = plan_grad(a.m, a.k, a.n, a.dtype);
    const uint64_t width = plan.width;
    const uint64_t gpitch = up(width, 64);
    const Plan& qx = plan.dx;
    const uint64_t xpart_rows = qx.split_rows, xpart_pitch = qx.part_pitch;
    for (const Plan& q : {plan.g, plan.dx, plan.dw, plan.dw_last}) KNNG_TRY(check_items(op, q));
    Carver c(ws);
    uint16_t* xs = c.take<uint16_t>(stage_elems(x, a.dtype));
    uint16_t* wst = needs_stage(w, a.dtype) ? c.take<uint16_t>(stage_elems(w, a.dtype)) : nullptr;
    float* coef = c.take<float>(a.m);
    float* lse2 = c.take<float>(a.m);
    const uint32_t row_blocks = static_cast<uint32_t>(std::min<uint64_t>(ceil_div(a.m, 256), 148));
    float* cmax = c.take<float>(row_blocks);
    float* rest = planes == 1 ? c.take<float>(a.m) : nullptr;
    uint16_t* g = c.take<uint16_t>(a.m * gpitch * planes);
    float* xpart = a.dx ? c.take<float>(qx.splits * xpart_rows * xpart_pitch) : nullptr;
    const uint64_t wpart_elems = a.dw ? std::max(plan.dw.part_elems(), plan.dw_last.part_elems()) : 0;
    float* wpart = wpart_elems ? c.take<float>(wpart_elems) : nullptr;
    if (need) {
        *need = c.at;
        return KNNG_GPU_OK;
    }
    KNNG_TRY(check_matrix(op, "x", a.x, a.m, a.k, a.ldx, a.dtype));
    KNNG_TRY(check_matrix(op, "w", a.w, a.n, a.k, a.ldw, a.dtype));
    if (a.dx) KNNG_TRY(check_matrix(op, "dx", a.dx, a.m, a.k, a.k, a.dtype));
    if (a.dw) KNNG_TRY(check_matrix(op, "dw", a.dw, a.n, a.k, a.k, a.dtype));
    if (!a.labels || !a.dloss || !a.lse)
        return fail(KNNG_GPU_INVALID_ARGUMENT, std::string(op) + ": labels, dloss or lse is NULL");
    KNNG_TRY(check_workspace(op, ws, ws_bytes, c.at));
    if (!a.dx && !a.dw) return KNNG_GPU_OK;
    int* err;
    KNNG_TRY(take_error(&err));
    const RowLabels labels{a.labels, a.labels_i64, static_cast<uint32_t>(a.n)};
    const GradRowsJob rows{a.dloss, a.lse, a.m, a.scale, a.labels, a.labels_i64, static_cast<uint32_t>(a.n), coef, lse2,
                           cmax, row_blocks};
    KNNG_TRY(prepare(a.dtype, stage_job(x, a.dtype, xs, labels), stage_job(w, a.dtype, wst), rows, st));
    const Operand ox = operand(x, a.dtype, xs), ow = operand(w, a.dtype, wst);
    // fp16 holds 2^14 g / max |dloss scale|: |g| <= 1 there, and the smallest
    // normal value 6e-5 then stands for 4e-9 instead of losing every p below it.
    const float gscale = a.dtype == KNNG_DTYPE_F16 ? 16384.0f : 1.0f;
    JoinParams join_w = {};
    for (uint64_t c0 = 0; c0 < a.n; c0 += width) {
        join_w = JoinParams{};
        const uint64_t cols = std::min(width, a.n - c0);
        const Operand wp{static_cast<const uint16_t*>(ow.ptr) + c0 * ow.ld, cols, ow.width, ow.ld, ow.plane};
        const Shape s1{a.m, cols, a.k, combos, f32, a.dtype == KNNG_DTYPE_BF16};
        const bool last = c0 + width >= a.n;
        const Plan q1 = last ? plan_grad_tiles(s1) : plan.g;
        ProductCall<1> call;
        KNNG_TRY(operand_maps(q1, ox, wp, kKK, operand_type(a.dtype), &call.map_a[0], &call.map_b[0]));
        ProductParams& p = call.p[0];
        p = base_params(s1, q1, ox, wp, kKK, a.dtype, err);
        p.scale2 = a.scale * 1.44269504088896f;
        p.labels = a.labels;
        p.labels_i64 = a.labels_i64;
        p.classes = static_cast<uint32_t>(a.n);
        p.class0 = static_cast<uint32_t>(c0);
        p.lse2 = lse2;
        p.coef = coef;
        p.alpha_dev = cmax;
        p.alpha_parts = row_blocks;
        p.grad_scale = gscale;
        p.grad_planes = planes;
        p.label_rest = rest;
        p.grad_pitch = static_cast<uint32_t>(gpitch);
        const uint64_t gld = gpitch * planes;
        const uint64_t gwidth = planes == 1 ? cols : gld;
        KNNG_TRY(make_map(&call.map_out[0], operand_type(a.dtype), g, gwidth, a.m, gld, 32, 32));
        call.map_pre[0] = call.map_out[0];
        KNNG_TRY(launch_product<kEpiGrad>(q1.cg, call, st));
        const Operand og{g, a.m, gwidth, gld, static_cast<uint32_t>(gpitch)};
        ProductCall<2> both;  // dx first: its items are the longer ones
        ProductCall<1> one;
        const bool merged = plan.merged && a.dx && a.dw;
        if (a.dx) {
            // Pieces add up in fp32, scaled when they are joined: the first one stores, the others add.
            const Shape sp{a.m, a.k, cols, combos, f32, a.dtype == KNNG_DTYPE_BF16};
            Plan qp = qx;
            qp.kblocks = static_cast<uint32_t>(ceil_div(cols, 64));
            qp.splits = std::min(qx.splits, qp.pieces());
            ProductParams px = base_params(sp, qp, og, wp, kKMN, a.dtype, err);
            px.out = xpart;
            px.out_type = kF32;
            px.out_tma = 1;
            px.accumulate = c0 > 0;
            px.split_rows = static_cast<uint32_t>(xpart_rows);
            CUtensorMap mga, mwb, mx;
            KNNG_TRY(operand_maps(qp, og, wp, kKMN, operand_type(a.dtype), &mga, &mwb));
            KNNG_TRY(make_map(&mx, KNNG_DTYPE_F32, xpart, xpart_pitch, qx.splits * xpart_rows, xpart_pitch, 32, 32));
            const auto set = [&](auto& call) {
                call.map_a[0] = mga;
                call.map_b[0] = mwb;
                call.map_out[0] = call.map_pre[0] = mx;
                call.p[0] = px;
            };
            if (merged) {
                set(both);
            } else {
                set(one);
                KNNG_TRY(launch_product<kEpiStore>(qp.cg, one, st));
            }
        }
        if (a.dw) {
            const Shape sw{cols, a.k, a.m, combos, f32, a.dtype == KNNG_DTYPE_BF16};
            const Plan& qw = last && c0 > 0 ? plan.dw_last : plan.dw;
            Tail t{static_cast<uint8_t*>(a.dw) + c0 * a.k * e, a.k, a.dtype};
            t.alpha = 1.0f / gscale;
            t.alpha_dev = cmax;
            t.alpha_parts = row_blocks;
            if (merged) {
                KNNG_TRY(set_store(both, 1, sw, qw, og, ox, kMNMN, a.dtype, t, wpart, &join_w, err));
                KNNG_TRY(launch_product<kEpiStore>(qw.cg, both, st));
            } else {
                KNNG_TRY(set_store(one, 0, sw, qw, og, ox, kMNMN, a.dtype, t, wpart, &join_w, err));
                KNNG_TRY(launch_product<kEpiStore>(qw.cg, one, st));
            }
        }
        // The last piece's joins wait for dx's.
        if (!last) KNNG_TRY(finish(SumsJob{}, join_w, JoinParams{}, st));
    }
    JoinParams j = {};
    if (a.dx) {
        j.part = xpart;
        j.splits = qx.splits;
        j.split_rows = xpart_rows;
        j.pitch = static_cast<uint32_t>(xpart_pitch);
        j.m = a.m;
        j.n = static_cast<uint32_t>(a.k);
        j.alpha = 1.0f / gscale;
        j.alpha_dev = cmax;
        j.alpha_parts = row_blocks;
        j.out = a.dx;
        j.ldo = a.k;
        j.out_type = a.dtype;
        j.labels = a.labels;
        j.labels_i64 = a.labels_i64;
        j.classes = static_cast<uint32_t>(a.n);
        // The label's entry of g carries most of a row's gradient: what its
        // rounding took is added back in fp32 (bf16, 8192 x 960 against 100,000
        // rows: dx off by 0.0017 of its norm instead of 0.0025).
        j.label_rest = rest;
        j.w = a.w;
        j.ldw = a.ldw;
        j.w_type = a.dtype;
        j.blocks = join_blocks(a.m, a.k);
    }
    return finish(SumsJob{}, join_w, j, st);
}

// ------------------------------------------------------------------ timeout test
knng_gpu_status selftest_product(int cg, uint64_t limit)
{
    struct Buffer {
        void* p = nullptr;
        ~Buffer() { cudaFree(p); }
    } rows, out;
    constexpr uint64_t kRows = 256, kWidth = 128;
    KNNG_CUDA(cudaMalloc(&rows.p, kRows * kWidth * 2));
    KNNG_CUDA(cudaMalloc(&out.p, kRows * kRows * 2));
    KNNG_CUDA(cudaMemset(rows.p, 0, kRows * kWidth * 2));
    int* err;
    KNNG_TRY(take_error(&err));
    const Shape s{kRows, kRows, kWidth, 1, false, true};
    const Operand a{rows.p, kRows, kWidth, kWidth, 0};
    ProductCall<1> call;
    KNNG_TRY(set_store(call, 0, s, tiles_of(s, cg, 128 * cg), a, a, kKK, KNNG_DTYPE_BF16,
                       Tail{out.p, kRows, KNNG_DTYPE_BF16}, nullptr, nullptr, err));
    call.p[0].wait_limit = static_cast<long long>(limit);
    call.p[0].test_mode = 1;
    KNNG_TRY(launch_product<kEpiStore>(cg, call, nullptr));
    KNNG_CUDA(cudaStreamSynchronize(nullptr));
    return take_error(&err);
}

// No exception leaves a C entry point.
template <class F>
knng_gpu_status guarded(F&& f)
{
    try {
        clear_last_error();
        return f();
    } catch (const std::bad_alloc&) {
        return KNNG_GPU_OUT_OF_MEMORY;
    } catch (...) {
        return KNNG_GPU_CUDA_ERROR;
    }
}

}  // namespace

extern "C" {

#define KNNG_LEARN_ENTRY(name)                                                                              \
    uint64_t knng_gpu_##name##_workspace_bytes(const knng_gpu_##name##_args* a)                             \
    {                                                                                                       \
        uint64_t need = 0;                                                                                  \
        if (!a) return 0;                                                                                   \
        const knng_gpu_status s = guarded([&] { return name##_run(*a, nullptr, 0, nullptr, &need); });      \
        return s == KNNG_GPU_OK ? need : 0;                                                                 \
    }                                                                                                       \
    knng_gpu_status knng_gpu_##name(const knng_gpu_##name##_args* a, void* d_workspace,                     \
                                    uint64_t workspace_bytes, void* stream)                                 \
    {                                                                                                       \
        return guarded([&] {                                                                                \
            if (!a) return fail(KNNG_GPU_INVALID_ARGUMENT, "knng::gpu::" #name ": args is NULL");           \
            return name##_run(*a, d_workspace, workspace_bytes, static_cast<cudaStream_t>(stream), nullptr); \
        });                                                                                                 \
    }

KNNG_LEARN_ENTRY(linear)
KNNG_LEARN_ENTRY(linear_backward)
KNNG_LEARN_ENTRY(softmax_xent)
KNNG_LEARN_ENTRY(softmax_xent_backward)

knng_gpu_status knng_gpu_selftest_product_wait(uint64_t wait_limit_cycles)
{
    return guarded([&]() -> knng_gpu_status {
        const knng_gpu_status pair = selftest_product(2, wait_limit_cycles);
        return pair == KNNG_GPU_TIMEOUT ? selftest_product(1, wait_limit_cycles) : pair;
    });
}

}  // extern "C"
