// product.cuh -- D = A B^T on the tensor cores with a fused epilogue: the one
// kernel behind the linear layer, the softmax loss over inner products and
// their gradients.
//
//   A is m x K, B is n x K. Either may lie in memory with K contiguous
//   ("K-major": rows of the operand) or with m / n contiguous ("MN-major": the
//   operand is the transpose of what is stored), so x w^T, dz w and dz^T x all
//   read the caller's rows as they lie, without a transposed copy.
//
// Operands are bf16 or fp16 with fp32 accumulation in TMEM. fp32 operands come
// as three bf16 planes (x = h + m + l, each the rounding of what the ones
// before left) and the product is the six plane products down to 2^-18 of the
// leading one, summed into the same accumulator; the three that are left out
// are below 2^-26 of it. Each plane of a K block is staged once and read by all
// the products that need it.
//
// Tile and roles. CG = 2: a CTA pair computes up to 256 x 256 with
// tcgen05.mma.cta_group::2; each CTA stages 128 rows of A and half the tile's
// rows of B per 64-wide K block, half of what two single-CTA tiles would read
// from L2. CG = 1: up to 128 x 128 by one CTA, for products with too few tiles
// to fill the GPU with pairs. Per CTA:
//   warp 0      TMA producer: as many stages as fit, 5 to 8
//   warp 1      TMEM allocation; UMMA issue (leader CTA, one lane)
//   warps 2-3   idle
//   warps 4 on  epilogue (8 or 16 warps): thread = one accumulator row, the
//               warps of a quarter of the rows take turns with the 32-column
//               chunks of a tile. Two accumulator buffers in TMEM: the
//               epilogue of a tile runs under the MMAs of the next one.
// Outputs leave through 4 KiB shared-memory boxes per warp and TMA stores
// (reduce-adds where a call accumulates), or by coalesced element stores where
// the output rows are not 16-byte aligned.
//
// What bounds it: the tensor cores (a K block of a pair's 256 x 256 tile takes
// them 512 cycles, and its 64 KiB come from L2 at about 60 bytes a cycle and
// SM), except where the epilogue's exponentials do (16 a cycle and SM). Measured
// on one B200: bf16 8192 x 4096 x 8192 372 us (1476 TFLOP/s, tensor pipe active
// 90%); softmax of 8192 x 960 against 100,000 rows 1048 us (1.50 PFLOP/s) when
// not throttled by power, 1240 us when it is; of 2048 x 128 against a million
// rows 548 us, the special-function units at 85%.
//
// Every wait is bounded: a role that gives up reports through *p.error (host
// memory), raises the abort flag of its CTA or pair, and all roles unwind.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace knng_b200 {

// Shared memory: a ring of stages (16 KiB of A and up to 16 KiB of B, a 64-wide
// K block of one plane) and the boxes through which the epilogue stores.
constexpr int kPkData = 229376;
constexpr int kPkSmem = kPkData + 512 + 1024;
constexpr int kPkMaxStages = 8;
constexpr int kPkStageA = 16384;

enum ElemType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4 };
enum Layout : int { kKK = 0, kKMN = 1, kMNMN = 2, kAnyLayout = 3 };  // how A and B are stored
enum Epilogue : int { kEpiStore = 0, kEpiSoftmax = 1, kEpiGrad = 2 };

struct ProductParams {
    uint32_t m, n;                 // rows and columns of D
    uint32_t tile_n;               // columns of a tile: a multiple of 32, at most 128 * CG
    uint32_t tiles_m, tiles_n;
    uint32_t splits;               // store: pieces of the K loop, each to its own rows of the output map
    uint32_t segments;             // softmax: pieces of the columns per row tile
    uint32_t items;                // work items = tiles_m * tiles_n * splits, or tiles_m * segments
    uint32_t kblocks;              // 64-wide K blocks of one plane
    uint32_t piece;                // K blocks (of every plane product) summed in TMEM before they leave it
    uint32_t pieces;               // ceil(kblocks / piece)
    uint32_t planes;               // 1, or 3 parts of split fp32 operands
    uint32_t plane_a, plane_b;     // columns from one plane to the next in the stored matrices
    int in_type;                   // kBF16 or kF16
    int layout;                    // Layout of A and B
    int* error;
    long long wait_limit;
    int test_mode;                 // 1: the producer withholds its first arrival (timeout test)
    // store
    int out_type;                  // ElemType
    int out_tma, pre_tma;          // TMA store possible; otherwise element stores through out / pre
    int accumulate;                // fp32 output: add to what is there
    void *out, *pre;
    uint64_t ldo, ldp;
    uint32_t split_rows;           // rows between the outputs of two splits
    const void* bias;              // of type aux_type
    const void* residual;
    uint64_t ldr;
    int aux_type;
    int bias_vec, residual_vec;    // they allow 16-byte loads
    int activation;
    float alpha;                   // D is scaled by alpha and, the last product of a call, by
    const float* alpha_dev;        // the largest of alpha_parts values there
    uint32_t alpha_parts;
    // softmax and gradient
    float scale2;                  // scale * log2(e)
    const void* labels;            // class of each row, int64 or int32; outside [0, classes) where it has none
    int labels_i64;
    uint32_t classes;
    uint32_t class0;               // class of column 0
    float2* part;                  // softmax: (max, sum) of row r, piece s, warp group h at [(groups s + h) * m + r]
    float* label_dot;              // softmax: x_r . w_label
    const float* lse2;             // gradient: lse * log2(e)
    const float* coef;             // gradient: dloss * scale / cmax, 0 for a row without label
    float grad_scale;              // gradient: power of two on the stored values
    uint32_t grad_planes, grad_pitch;
    float* label_rest;             // gradient: what rounding took from the label's entry (one plane)
};

// N products in one launch, the items of the second after those of the first.
template <int N>
struct ProductCall {
    CUtensorMap map_a[N], map_b[N], map_out[N], map_pre[N];
    ProductParams p[N];
};

// ---------------------------------------------------------------- PTX of this kernel
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                              uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// Descriptor of an MN-major operand staged as blocks of 64 (MN) x 64 (K): rows
// of 128 bytes along MN, one per K index, 128-byte swizzle. Eight K rows are
// 1024 bytes apart (stride offset), the next 64 MN values 8 KiB (leading
// offset).
__device__ __forceinline__ uint64_t umma_desc_mn_sw128(uint32_t saddr)
{
    uint64_t desc = 0;
    desc |= static_cast<uint64_t>((saddr >> 4) & 0x3FFFu);
    desc |= static_cast<uint64_t>(8192u >> 4) << 16;
    desc |= static_cast<uint64_t>(1024u >> 4) << 32;
    desc |= static_cast<uint64_t>(1u) << 46;
    desc |= static_cast<uint64_t>(2u) << 61;
    return desc;
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* smem, int32_t x, int32_t y)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(smem_u32(smem))
                 : "memory");
}

__device__ __forceinline__ void tma_reduce_add_2d(const CUtensorMap* map, const void* smem, int32_t x, int32_t y)
{
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                     reinterpret_cast<uint64_t>(map)),
                 "r"(x), "r"(y), "r"(smem_u32(smem))
                 : "memory");
}

__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void bulk_wait_read()
{
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Two fp32 operations per instruction.
__device__ __forceinline__ uint64_t pair_f32(float a, float b)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair_f32(uint64_t v)
{
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// ---------------------------------------------------------------- elementwise pieces
__device__ __forceinline__ uint32_t pack2(float a, float b, int type)
{
    uint32_t r;
    if (type == kBF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        memcpy(&r, &v, 4);
    } else {
        const __half2 v = __floats2half2_rn(a, b);
        memcpy(&r, &v, 4);
    }
    return r;
}

__device__ __forceinline__ float load_elem(const void* p, uint64_t i, int type)
{
    if (type == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    if (type == kF16) return __half2float(static_cast<const __half*>(p)[i]);
    return static_cast<const float*>(p)[i];
}

__device__ __forceinline__ void store_elem(void* p, uint64_t i, float v, int type)
{
    if (type == kBF16)
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else if (type == kF16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<float*>(p)[i] = v;
}

// Two 16-bit values of a word as floats.
__device__ __forceinline__ float2 unpack2(uint32_t w, int type)
{
    if (type == kBF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    __half2 h;
    memcpy(&h, &w, 4);
    return __half22float2(h);
}

__device__ __forceinline__ float rcp_approx(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint64_t both(float c) { return pair_f32(c, c); }
__device__ __forceinline__ uint64_t exp2_pair(uint64_t x)
{
    const float2 f = unpair_f32(x);
    return pair_f32(exp2_approx(f.x), exp2_approx(f.y));
}
__device__ __forceinline__ uint64_t rcp_pair(uint64_t x)
{
    const float2 f = unpair_f32(x);
    return pair_f32(rcp_approx(f.x), rcp_approx(f.y));
}

// The activations and their slopes, two values at a time: the epilogues that
// use them are bound by issue slots.

// sigmoid(v) = 1 / (1 + e^-v); e^-v overflows to +inf for very negative v,
// where the quotient is 0 as it should be.
__device__ __forceinline__ uint64_t sigmoid2(uint64_t v)
{
    return rcp_pair(add2(exp2_pair(mul2(v, both(-1.44269504f))), both(1.0f)));
}

// The normal distribution function Phi(z) and *bell = e^(-z^2 / 2), by
// Abramowitz and Stegun 7.1.26: erfc(x) = (a1 t + ... + a5 t^5) e^(-x^2) with
// t = 1 / (1 + 0.3275911 x), off by at most 1.5e-7 for x = |z| / sqrt 2 >= 0.
// No branch, and the slope needs the same exponential. q is Phi(-|z|) =
// erfc(x) / 2, and Phi(z) = 1/2 + (1/2 - q) with the sign of z.
__device__ __forceinline__ uint64_t normal_cdf2(uint64_t z, uint64_t* bell)
{
    const uint64_t e = exp2_pair(mul2(mul2(z, z), both(-0.72134752f)));
    const uint64_t t = rcp_pair(fma2(z & 0x7FFFFFFF7FFFFFFFull, both(0.23164189f), both(1.0f)));
    uint64_t q = fma2(t, both(0.530702715f), both(-0.726576014f));  // half the coefficients
    q = fma2(t, q, both(0.710706871f));
    q = fma2(t, q, both(-0.142248368f));
    q = fma2(t, q, both(0.127414796f));
    q = mul2(mul2(q, t), e);
    *bell = e;
    const uint64_t r = fma2(q, both(-1.0f), both(0.5f));
    return add2((r & 0x7FFFFFFF7FFFFFFFull) | (z & 0x8000000080000000ull), both(0.5f));
}

template <int ACT>
__device__ __forceinline__ uint64_t act2(uint64_t z)
{
    if constexpr (ACT == kActRelu) {
        const float2 f = unpair_f32(z);
        return pair_f32(f.x < 0.0f ? 0.0f : f.x, f.y < 0.0f ? 0.0f : f.y);  // NaN stays NaN
    }
    if constexpr (ACT == kActGelu) {
        uint64_t bell;
        return mul2(z, normal_cdf2(z, &bell));
    }
    // 0.5 (1 + tanh u) = sigmoid(2 u), 2 u = z (c + 0.044715 c z^2), c = 2 sqrt(2/pi).
    if constexpr (ACT == kActGeluTanh)
        return mul2(z, sigmoid2(mul2(z, fma2(mul2(z, z), both(0.0713548163f), both(1.59576912f)))));
    if constexpr (ACT == kActSilu) return mul2(z, sigmoid2(z));
    return z;
}

template <int ACT>
__device__ __forceinline__ uint64_t slope2(uint64_t z)
{
    if constexpr (ACT == kActRelu) {
        const float2 f = unpair_f32(z);
        return pair_f32(f.x > 0.0f ? 1.0f : 0.0f, f.y > 0.0f ? 1.0f : 0.0f);
    }
    if constexpr (ACT == kActGelu) {
        uint64_t bell;
        const uint64_t phi = normal_cdf2(z, &bell);
        return fma2(mul2(z, both(0.39894228f)), bell, phi);
    }
    if constexpr (ACT == kActGeluTanh) {
        const uint64_t zz = mul2(z, z);
        const uint64_t s = sigmoid2(mul2(z, fma2(zz, both(0.0713548163f), both(1.59576912f))));
        const uint64_t du = fma2(zz, both(0.214064449f), both(1.59576912f));
        // s + z s (1 - s) du
        return fma2(mul2(mul2(z, s), fma2(s, both(-1.0f), both(1.0f))), du, s);
    }
    if constexpr (ACT == kActSilu) {
        const uint64_t s = sigmoid2(z);
        return mul2(s, fma2(z, fma2(s, both(-1.0f), both(1.0f)), both(1.0f)));
    }
    return both(1.0f);
}

template <int ACT>
__device__ __forceinline__ float act_f(float z)
{
    return unpair_f32(act2<ACT>(both(z))).x;
}

// One value of the linear epilogue (shared with the join of split products).
__device__ __forceinline__ float act_dyn(float z, int act)
{
    switch (act) {
        case kActRelu: return act_f<kActRelu>(z);
        case kActGelu: return act_f<kActGelu>(z);
        case kActGeluTanh: return act_f<kActGeluTanh>(z);
        case kActSilu: return act_f<kActSilu>(z);
        default: return z;
    }
}

// 32 values as 16 words of two.
__device__ __forceinline__ void pack32(const float* v, uint32_t* w, int type)
{
    if (type == kBF16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], kBF16);
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] = pack2(v[2 * j], v[2 * j + 1], kF16);
    }
}

// Adds 32 consecutive 16-bit values.
__device__ __forceinline__ void add_words(float* v, const uint4* src, int type)
{
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint4 q = src[j];
        w[4 * j] = q.x, w[4 * j + 1] = q.y, w[4 * j + 2] = q.z, w[4 * j + 3] = q.w;
    }
    if (type == kBF16) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float2 f = unpack2(w[j], kBF16);
            const float2 r = unpair_f32(add2(pair_f32(v[2 * j], v[2 * j + 1]), pair_f32(f.x, f.y)));
            v[2 * j] = r.x;
            v[2 * j + 1] = r.y;
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float2 f = unpack2(w[j], kF16);
            const float2 r = unpair_f32(add2(pair_f32(v[2 * j], v[2 * j + 1]), pair_f32(f.x, f.y)));
            v[2 * j] = r.x;
            v[2 * j + 1] = r.y;
        }
    }
}

template <int ACT>
__device__ __forceinline__ void act_all(float* v)
{
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float2 r = unpair_f32(act2<ACT>(pair_f32(v[i], v[i + 1])));
        v[i] = r.x;
        v[i + 1] = r.y;
    }
}

// Class of a row, -1 where it has none.
__device__ __forceinline__ int32_t load_label(const void* labels, int i64, uint64_t row, uint32_t classes)
{
    const int64_t y = i64 ? static_cast<const int64_t*>(labels)[row]
                          : static_cast<int64_t>(static_cast<const int32_t*>(labels)[row]);
    return y >= 0 && y < static_cast<int64_t>(classes) ? static_cast<int32_t>(y) : -1;
}

// The largest of n values >= 0 (0 if there are none), in every lane of a warp.
__device__ __forceinline__ float warp_largest(const float* v, uint32_t n)
{
    float big = 0.0f;
    for (uint32_t i = threadIdx.x & 31; i < n; i += 32) big = fmaxf(big, v[i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, o));
    return big;
}

// ---------------------------------------------------------------- schedule
struct Item {
    uint32_t tm, n0, n1, p0, p1, split, segment;  // row tile, column tiles, K pieces
};

template <int EPI>
__device__ __forceinline__ Item decode_item(const ProductParams& p, uint32_t i)
{
    Item t;
    if constexpr (EPI == kEpiSoftmax) {
        // Items next to each other walk the same columns for different row
        // tiles, so B is read from HBM once.
        t.segment = i / p.tiles_m;
        t.tm = i % p.tiles_m;
        t.n0 = static_cast<uint32_t>(uint64_t(t.segment) * p.tiles_n / p.segments);
        t.n1 = static_cast<uint32_t>(uint64_t(t.segment + 1) * p.tiles_n / p.segments);
        t.split = 0;
        t.p0 = 0;
        t.p1 = p.pieces;
    } else {
        // Bands of 8 row tiles, walked column tile by column tile: the units
        // that run together share A and B tiles in L2.
        const uint32_t tiles = p.tiles_m * p.tiles_n;
        t.split = i / tiles;
        const uint32_t r = i % tiles;
        const uint32_t band = r / (8 * p.tiles_n);
        const uint32_t rows = min(8u, p.tiles_m - band * 8);
        const uint32_t q = r - band * 8 * p.tiles_n;
        t.tm = band * 8 + q % rows;
        t.n0 = q / rows;
        t.n1 = t.n0 + 1;
        t.segment = 0;
        t.p0 = static_cast<uint32_t>(uint64_t(t.split) * p.pieces / p.splits);
        t.p1 = static_cast<uint32_t>(uint64_t(t.split + 1) * p.pieces / p.splits);
    }
    return t;
}

// ---------------------------------------------------------------- kernel
// Epilogue warps: 16, or 8 where sums over long K need the registers and for
// the softmax of single CTAs, whose warps take two chunks at once. With 8, two
// warps per scheduler leave every latency of an epilogue exposed: 2048 x 128
// against a million rows took 621 us instead of 572, a gelu layer of 100,000 x
// 784 -> 1024 249 us instead of 189.
__host__ __device__ constexpr int pk_epi_warps(int cg, int epi, bool longk)
{
    return longk || (cg == 1 && epi == kEpiSoftmax) ? 8 : 16;
}
// Boxes of 32 rows x 32 columns. 16 warps have two for 16-bit values (an fp32
// box takes both), 8 warps two of those or one of fp32: the ring gets the rest,
// which six plane products of fp32 operands need most, three stages at a time.
__host__ __device__ constexpr int pk_box_bytes(int cg, int epi, bool longk)
{
    return epi == kEpiSoftmax ? 0 : 4096 * pk_epi_warps(cg, epi, longk);
}
__host__ __device__ constexpr int pk_threads(int cg, int epi, bool longk) { return 128 + 32 * pk_epi_warps(cg, epi, longk); }
// Registers a thread: what the launch gives, and the split after setmaxnreg
// between the first warpgroup and those of the epilogue. The split never sums
// to more than the launch gave: 72 + 2 * 216 = 3 * 168, 64 + 4 * 104 = 5 * 96.
__host__ __device__ constexpr int pk_launch_regs(int warps) { return warps == 8 ? 168 : 96; }
__host__ __device__ constexpr int pk_issue_regs(int warps) { return warps == 8 ? 72 : 64; }
__host__ __device__ constexpr int pk_epi_regs(int warps) { return warps == 8 ? 216 : 104; }

// LONG: an item may have several K pieces, whose sums are added in registers.
// N = 2: the two products of a backward pass, which need only part of the GPU
// each when they are small and an uneven last round when they are not; plain
// stores.
// LAY: how the operands lie, or kAnyLayout to take it from each product (known
// at compile time it saves the issuing threads 5 to 10 % of a long product).
template <int CG, int EPI, bool LONG, int N, int LAY>
__global__ void __launch_bounds__(pk_threads(CG, EPI, LONG), 1)
    product_kernel(const __grid_constant__ ProductCall<N> call)
{
    constexpr int EW = pk_epi_warps(CG, EPI, LONG);
    // Softmax with 16 warps: eight for each of the two accumulator buffers, so
    // that one half exponentiates while the other waits, loads and looks for
    // maxima (2048 x 128 against a million rows: 583 -> 558 us; stores gain
    // nothing, a gelu layer of 100,000 x 784 -> 1024 took 203 us instead of 189).
    constexpr int kSets = EPI == kEpiSoftmax && EW == 16 ? 2 : 1;
    constexpr int kGroups = EW / 4 / kSets;  // warps that share a quarter of the rows of a tile
    constexpr uint32_t kBufCols = 128 * CG;  // TMEM columns of an accumulator buffer
    constexpr uint32_t kTmemCols = 2 * kBufCols;
    const uint32_t items0 = call.p[0].items;
    const uint32_t items = items0 + (N == 2 ? call.p[N - 1].items : 0u);
    const long long wait_limit = call.p[0].wait_limit;
    constexpr int kBoxBytes = pk_box_bytes(CG, EPI, LONG);
    // Bytes of B that a CTA stages for a K block, and the ring for the widest product.
    const auto b_bytes_of = [&](const ProductParams& p) -> uint32_t {
        const int lay = LAY == kAnyLayout ? p.layout : LAY;
        const uint32_t cols = p.tile_n / CG;
        return lay == kKK ? cols * 128u : (cols > 64 ? 16384u : 8192u);
    };
    uint32_t stage_bytes = kPkStageA + b_bytes_of(call.p[0]);
    if constexpr (N == 2) stage_bytes = max(stage_bytes, kPkStageA + b_bytes_of(call.p[N - 1]));
    const uint32_t stages = min(static_cast<uint32_t>(kPkData - kBoxBytes) / stage_bytes, static_cast<uint32_t>(kPkMaxStages));
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* stage_base = smem;
    uint8_t* boxes = smem + kPkData - kBoxBytes;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPkData);
    uint64_t* full = bars;        // [kPkMaxStages] leader: bytes of both CTAs landed
    uint64_t* empty = bars + 8;   // [kPkMaxStages] both: MMAs that read the stage are done
    uint64_t* tfull = bars + 16;  // [2] both: accumulator ready
    uint64_t* tempty = bars + 18; // [2] leader: accumulator read by the epilogue warps of both CTAs
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 20);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 21);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t cta = CG == 2 ? (cluster_ctarank() & 1u) : 0u;
    const bool leader = cta == 0;
    const uint32_t unit = blockIdx.x / CG;
    const uint32_t units = gridDim.x / CG;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kPkMaxStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], CG * EW / kSets);
        }
        *abort_flag = 0;
        fence_barrier_init();
        for (int i = 0; i < N; ++i) {
            prefetch_tensormap(&call.map_a[i]);
            prefetch_tensormap(&call.map_b[i]);
        }
    }
    if (warp == 1) {
        if constexpr (CG == 2)
            tmem_alloc_pair(tmem_slot, kTmemCols);
        else
            tmem_alloc(tmem_slot, kTmemCols);
    }
    tc_fence_before();
    if constexpr (CG == 2)
        cluster_sync_all();
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    previous_done();

    auto abort_all = [&]() {
        *call.p[0].error = 1;
        __threadfence_system();
        *abort_flag = 1;
        if constexpr (CG == 2) st_cluster_u32(mapa_shared(smem_u32(const_cast<int*>(abort_flag)), cta ^ 1u), 1u);
    };

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pk_issue_regs(EW)));
        if (lane == 0) {
            const uint32_t full_leader = CG == 2 ? mapa_shared(smem_u32(full), 0u) : 0u;
            uint32_t stage = 0, phase = 0, issued = 0;
            bool ok = true;
            for (uint32_t i = unit; ok && i < items; i += units) {
                const int which = N == 2 && i >= items0;
                const ProductParams& p = call.p[which];
                const CUtensorMap* map_a = &call.map_a[which];
                const CUtensorMap* map_b = &call.map_b[which];
                const int lay = LAY == kAnyLayout ? p.layout : LAY;
                const bool a_mn = lay == kMNMN, b_mn = lay != kKK;
                const uint32_t bn_tile = p.tile_n, bn_cta = bn_tile / CG;  // rows of B that this CTA stages
                const uint32_t tx = CG * (kPkStageA + b_bytes_of(p));
                const uint32_t planes = p.planes, plane_a = p.plane_a, plane_b = p.plane_b;
                const Item t = decode_item<EPI>(p, which ? i - items0 : i);
                const int32_t am = static_cast<int32_t>(t.tm * (128 * CG) + cta * 128);
                for (uint32_t tn = t.n0; ok && tn < t.n1; ++tn) {
                    const int32_t bn = static_cast<int32_t>(tn * bn_tile + cta * bn_cta);
                    const uint32_t kb1 = min(t.p1 * p.piece, p.kblocks);
                    uint32_t kb = t.p0 * p.piece, plane = planes;
                    while (kb < kb1) {
                        const int32_t k = static_cast<int32_t>(kb * 64);
                        --plane;  // the smallest plane of a K block first
                        const int32_t pa = static_cast<int32_t>(plane * plane_a);
                        const int32_t pb = static_cast<int32_t>(plane * plane_b);
                        if (plane == 0) {
                            plane = planes;
                            ++kb;
                        }
                        ok = mbar_wait(&empty[stage], phase ^ 1, abort_flag, wait_limit);
                        if (!ok) break;
                        uint8_t* sa = stage_base + stage * stage_bytes;
                        uint8_t* sb = sa + kPkStageA;
                        if (leader && !(call.p[0].test_mode == 1 && issued == 0)) mbar_arrive_expect_tx(&full[stage], tx);
                        auto load = [&](uint8_t* dst, const CUtensorMap* map, int32_t x, int32_t y) {
                            if constexpr (CG == 2)
                                tma_load_2d_pair(dst, map, x, y, full_leader + stage * 8);
                            else
                                tma_load_2d(dst, map, x, y, &full[stage]);
                        };
                        if (a_mn) {
                            load(sa, map_a, pa + am, k);
                            load(sa + 8192, map_a, pa + am + 64, k);
                        } else {
                            load(sa, map_a, pa + k, am);
                        }
                        if (b_mn) {
                            load(sb, map_b, pb + bn, k);
                            if (bn_cta > 64) load(sb + 8192, map_b, pb + bn + 64, k);
                        } else {
                            load(sb, map_b, pb + k, bn);
                        }
                        ++issued;
                        if (++stage == stages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    }
                }
            }
            if (!ok) {
                abort_all();
                // Copies in flight land before the CTA's memory goes away: the
                // last use of each stage, a bounded wait each.
                if (leader) {
                    for (uint32_t s = 0; s < stages; ++s) {
                        if (issued <= s) break;
                        const uint32_t uses = (issued - s - 1) / stages;  // 0-based index of its last use
                        (void)mbar_wait_drain(&full[s], uses & 1, wait_limit / 8);
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ------------------------------------------------ UMMA issuer
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pk_issue_regs(EW)));
        if (leader && lane == 0) {
            const uint32_t s0 = smem_u32(stage_base);
            uint32_t stage = 0, phase = 0, acc = 0;
            bool ok = true;
            for (uint32_t i = unit; ok && i < items; i += units) {
                const int which = N == 2 && i >= items0;
                const ProductParams& p = call.p[which];
                const int lay = LAY == kAnyLayout ? p.layout : LAY;
                const bool a_mn = lay == kMNMN, b_mn = lay != kKK;
                const uint32_t fmt = p.in_type == kBF16 ? 1u : 0u;
                const uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (a_mn ? 1u << 15 : 0u) |
                                       (b_mn ? 1u << 16 : 0u) | ((p.tile_n >> 3) << 17) |
                                       (static_cast<uint32_t>((128 * CG) >> 4) << 24);
                const uint64_t a0 = a_mn ? umma_desc_mn_sw128(s0) : umma_desc_sw128(s0);
                const uint64_t b0 = b_mn ? umma_desc_mn_sw128(s0 + kPkStageA) : umma_desc_sw128(s0 + kPkStageA);
                const uint64_t ka = a_mn ? 2048 >> 4 : 2;  // 16 of K: 16 rows of 128 bytes, or 32 bytes
                const uint64_t kb = b_mn ? 2048 >> 4 : 2;
                const uint32_t planes = p.planes;
                const Item t = decode_item<EPI>(p, which ? i - items0 : i);
                const uint32_t pieces = (t.n1 - t.n0) * (t.p1 - t.p0);
                for (uint32_t q = 0; ok && q < pieces; ++q, ++acc) {
                    const uint32_t piece = t.p0 + q % (t.p1 - t.p0);
                    const uint32_t blocks = min((piece + 1) * p.piece, p.kblocks) - piece * p.piece;
                    const uint32_t buf = acc & 1u;
                    ok = mbar_wait_sleep(&tempty[buf], ((acc >> 1) & 1u) ^ 1u, abort_flag, wait_limit);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t d = tmem_base + buf * kBufCols;
                    auto stage_ready = [&]() {
                        const bool r = mbar_wait_sleep(&full[stage], phase, abort_flag, wait_limit);
                        tc_fence_after();
                        return r;
                    };
                    auto next_stage = [&]() {
                        if (++stage == stages) {
                            stage = 0;
                            phase ^= 1;
                        }
                    };
                    // One K block of stage sa's A against stage sb's B.
                    auto multiply = [&](uint32_t sa, uint32_t sb, bool more) {
                        const uint64_t ad = a0 + sa * (stage_bytes >> 4);
                        const uint64_t bd = b0 + sb * (stage_bytes >> 4);
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const uint32_t add = more || ks > 0 ? 1u : 0u;
                            if constexpr (CG == 2)
                                umma_f16_pair(d, ad + ks * ka, bd + ks * kb, idesc, add);
                            else
                                umma_f16(d, ad + ks * ka, bd + ks * kb, idesc, add);
                        }
                    };
                    auto stage_done = [&](uint32_t s) {
                        if constexpr (CG == 2)
                            umma_commit_pair(&empty[s]);
                        else
                            umma_commit(&empty[s]);
                    };
                    if (planes == 1) {
                        for (uint32_t kk = 0; kk < blocks; ++kk) {
                            ok = stage_ready();
                            if (!ok) break;
                            multiply(stage, stage, kk > 0);
                            stage_done(stage);
                            next_stage();
                        }
                    } else {
                        // Planes l, m, h of a K block, the small products first:
                        // each addition costs a truncation of what is there.
                        // A piece is one K block here, so the accumulator holds
                        // only small sums until the last product.
                        for (uint32_t kk = 0; kk < blocks; ++kk) {
                            uint32_t at[3];
#pragma unroll
                            for (int plane = 2; plane >= 0; --plane) {
                                if (ok) ok = stage_ready();
                                at[plane] = stage;
                                next_stage();
                            }
                            if (!ok) break;
                            multiply(at[0], at[2], kk > 0);
                            multiply(at[2], at[0], true);
                            stage_done(at[2]);
                            multiply(at[1], at[1], true);
                            multiply(at[1], at[0], true);
                            multiply(at[0], at[1], true);
                            stage_done(at[1]);
                            multiply(at[0], at[0], true);
                            stage_done(at[0]);
                        }
                    }
                    if (!ok) break;
                    if constexpr (CG == 2)
                        umma_commit_pair(&tfull[buf]);
                    else
                        umma_commit(&tfull[buf]);
                }
            }
            if (!ok) abort_all();
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------ epilogue
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(pk_epi_regs(EW)));
        const int e = warp - 4;
        const uint32_t quarter = warp & 3;
        const uint32_t group = (e >> 2) % kGroups;
        const uint32_t set = (e >> 2) / kGroups;
        // 32-column chunks of this warp: number group, group + kGroups, ...
        constexpr int kMaxChunks = 4 * CG / kGroups;
        constexpr uint32_t kStep = 32 * kGroups;  // columns from one to the next
        int chunks = 0;  // of the current item
        const ProductParams* at_work = &call.p[0];  // the current item's product
        uint8_t* box = boxes + e * 4096;
        uint32_t nbox = 0;  // boxes sent: picks the buffer
        const uint32_t tempty_leader = CG == 2 ? mapa_shared(smem_u32(tempty), 0u) : 0u;
        const uint32_t lane_base = tmem_base + ((quarter * 32u) << 16) + group * 32;
        uint32_t acc = 0;
        bool ok = true;

        // The buffer of the next box, once the store that read it is done: two
        // 16-bit boxes take turns, an fp32 box takes the room of both.
        bool whole = false;  // the last box did
        auto next_box = [&](bool f32 = false) -> uint8_t* {
            uint8_t* b = box + (f32 ? 0u : (nbox & 1u) * 2048u);
            ++nbox;
            if (lane == 0) {
                if (f32 || whole)
                    bulk_wait_read<0>();
                else
                    bulk_wait_read<1>();
            }
            whole = f32;
            __syncwarp();
            return b;
        };
        // This thread's row of a box, swizzled as the TMA maps expect: 32 fp32
        // values in 128-byte rows, or 32 16-bit values (16 words) in 64-byte rows.
        auto put_f32 = [&](uint8_t* b, const float* v) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                *reinterpret_cast<uint4*>(b + lane * 128 + ((j ^ (lane & 7)) << 4)) =
                    make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                               __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
        };
        auto put_words = [&](uint8_t* b, const uint32_t* w) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<uint4*>(b + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
                    make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        };
        auto send = [&](const uint8_t* b, const CUtensorMap* map, uint32_t x, uint32_t y, bool add) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                if (add)
                    tma_reduce_add_2d(map, b, static_cast<int32_t>(x), static_cast<int32_t>(y));
                else
                    tma_store_2d(map, b, static_cast<int32_t>(x), static_cast<int32_t>(y));
                bulk_commit();
            }
            __syncwarp();
        };
        // Element stores of a box to rows that TMA cannot write.
        auto copy_out = [&](const uint8_t* b, void* dst, uint64_t ld, int esize, uint32_t row0, uint32_t col0) {
            const ProductParams& p = *at_work;
            __syncwarp();
            const int rows = row0 < p.m ? static_cast<int>(min(32u, p.m - row0)) : 0;
            if (col0 + lane < p.n) {
                // A row at a time over the lanes, eight rows in flight.
                const uint64_t first = row0 * ld + col0 + lane;
#pragma unroll 1
                for (int r = 0; r < rows; r += 8) {
                    uint32_t v[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int q = r + i;  // rows past the last hold values too, only nobody stores them
                        if (esize == 2)
                            v[i] = *reinterpret_cast<const uint16_t*>(
                                b + q * 64 + (((lane >> 3) ^ ((q >> 1) & 3)) << 4) + (lane & 7) * 2);
                        else
                            v[i] = *reinterpret_cast<const uint32_t*>(
                                b + q * 128 + (((lane >> 2) ^ (q & 7)) << 4) + (lane & 3) * 4);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (r + i >= rows) break;
                        const uint64_t at = first + (r + i) * ld;
                        if (esize == 2)
                            static_cast<uint16_t*>(dst)[at] = static_cast<uint16_t>(v[i]);
                        else
                            static_cast<uint32_t*>(dst)[at] = v[i];
                    }
                }
            }
            __syncwarp();
            if (lane == 0) bulk_commit();  // an empty group: the buffers keep taking turns
        };
        auto issue = [&](uint32_t buf, int i, float* v) {
            tmem_ld_32cols(lane_base + buf * kBufCols + i * kStep, reinterpret_cast<int32_t*>(v));
        };
        auto arrived = [&](float* v) { tmem_ld_wait_n<32>(reinterpret_cast<int32_t*>(v)); };
        auto release = [&](uint32_t buf) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CG == 2)
                    mbar_arrive_remote(tempty_leader + buf * 8);
                else
                    mbar_arrive(&tempty[buf]);
            }
        };
        auto wait_acc = [&](uint32_t& buf) -> bool {
            buf = acc & 1u;
            if (!mbar_wait(&tfull[buf], (acc >> 1) & 1u, abort_flag, wait_limit)) return false;
            ++acc;
            tc_fence_after();
            return true;
        };
        // The tensor cores add into TMEM by truncation, which over a long K
        // pulls every sum towards zero by parts in 10^5: K is summed there in
        // pieces, and the pieces are added in registers, rounded to nearest.
        // This warp's chunks of the next tile, summed over its pieces.
        auto sum_pieces = [&](uint32_t pieces, float* sums) -> bool {
#pragma unroll
            for (int j = 0; j < 32 * kMaxChunks; ++j) sums[j] = 0.0f;
            for (uint32_t q = 0; q < pieces; ++q) {
                uint32_t buf;
                if (!wait_acc(buf)) return false;
                // Two chunks in flight at a time; the buffer goes back as soon
                // as the last ones are in registers.
#pragma unroll
                for (int i = 0; i < kMaxChunks; i += 2) {
                    float v[64];
                    if (i < chunks) issue(buf, i, v);
                    if (i + 1 < chunks) issue(buf, i + 1, v + 32);
                    arrived(v);
                    tie32(reinterpret_cast<int32_t*>(v + 32));
                    if (i + 2 >= kMaxChunks) release(buf);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        if (i + h >= chunks) break;
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            float* s2 = sums + 32 * (i + h) + j;
                            const float2 r = unpair_f32(add2(pair_f32(s2[0], s2[1]), pair_f32(v[32 * h + j], v[32 * h + j + 1])));
                            s2[0] = r.x;
                            s2[1] = r.y;
                        }
                    }
                }
            }
            return true;
        };
        // Calls f(v, chunk) for this warp's chunks of the next tile.
        auto for_tile = [&](uint32_t pieces, auto&& f) -> bool {
            if constexpr (!LONG) {
                uint32_t buf;
                if (!wait_acc(buf)) return false;
                if (chunks == 0) release(buf);
#pragma unroll 1
                for (int i = 0; i < chunks; ++i) {
                    float v[32];
                    issue(buf, i, v);
                    arrived(v);
                    if (i + 1 == chunks) release(buf);
                    f(v, i);
                }
            } else {
                float sums[32 * kMaxChunks];
                if (!sum_pieces(pieces, sums)) return false;
#pragma unroll
                for (int i = 0; i < kMaxChunks; ++i)
                    if (i < chunks) f(sums + 32 * i, i);
            }
            return true;
        };

        // Only the last product of a call is scaled by it.
        const ProductParams& scaled = call.p[N - 1];
        const float largest = scaled.alpha_dev ? warp_largest(scaled.alpha_dev, scaled.alpha_parts) : 1.0f;
        for (uint32_t it = unit; ok && it < items; it += units) {
            const int which = N == 2 && it >= items0;
            if constexpr (N == 2) at_work = &call.p[which];
            const ProductParams& p = call.p[which];
            const CUtensorMap* map_out = &call.map_out[which];
            const uint32_t bn_tile = p.tile_n;
            chunks = static_cast<int>((bn_tile / 32 + kGroups - 1 - group) / kGroups);
            const Item t = decode_item<EPI>(p, which ? it - items0 : it);
            const uint32_t row0 = t.tm * (128 * CG) + cta * 128 + quarter * 32;
            const uint32_t row = row0 + lane;
            const bool live = row < p.m;

            if constexpr (EPI == kEpiStore) {
                const float alpha = which == N - 1 ? p.alpha * largest : p.alpha;
                const uint32_t col_base = t.n0 * bn_tile + group * 32;
                const uint32_t out_row0 = row0 + t.split * p.split_rows;
                ok = for_tile(t.p1 - t.p0, [&](float* v, int i) {
                    const uint32_t col = col_base + i * kStep;
                    if (row0 >= p.m || col >= p.n) return;  // nobody reads what lies there
                    if (alpha != 1.0f) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] *= alpha;
                    }
                    if (N == 1 && p.bias) {
                        if (p.bias_vec && col + 32 <= p.n) {
                            if (p.aux_type == kF32) {
                                const float4* q4 = reinterpret_cast<const float4*>(static_cast<const float*>(p.bias) + col);
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float4 q = q4[j];
                                    v[4 * j] += q.x;
                                    v[4 * j + 1] += q.y;
                                    v[4 * j + 2] += q.z;
                                    v[4 * j + 3] += q.w;
                                }
                            } else {
                                add_words(v, reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.bias) + col),
                                          p.aux_type);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (col + j < p.n) v[j] += load_elem(p.bias, col + j, p.aux_type);
                        }
                    }
                    if (N == 1 && p.pre) {
                        // The value before the activation, rounded to the inputs' type.
                        uint8_t* b = next_box(p.aux_type == kF32);
                        if (p.aux_type == kF32) {
                            put_f32(b, v);
                        } else {
                            uint32_t w[16];
                            pack32(v, w, p.aux_type);
                            put_words(b, w);
                        }
                        if (p.pre_tma)
                            send(b, &call.map_pre[0], col, row0, false);
                        else
                            copy_out(b, p.pre, p.ldp, p.aux_type == kF32 ? 4 : 2, row0, col);
                    }
                    switch (N == 1 ? p.activation : 0) {
                        case kActRelu: act_all<kActRelu>(v); break;
                        case kActGelu: act_all<kActGelu>(v); break;
                        case kActGeluTanh: act_all<kActGeluTanh>(v); break;
                        case kActSilu: act_all<kActSilu>(v); break;
                        default: break;
                    }
                    if (N == 1 && p.residual && live) {
                        const uint64_t at = row * p.ldr + col;
                        if (p.residual_vec && col + 32 <= p.n) {
                            if (p.aux_type == kF32) {
                                const float4* r4 = reinterpret_cast<const float4*>(static_cast<const float*>(p.residual) + at);
#pragma unroll
                                for (int j = 0; j < 8; ++j) {
                                    const float4 q = r4[j];
                                    v[4 * j] += q.x;
                                    v[4 * j + 1] += q.y;
                                    v[4 * j + 2] += q.z;
                                    v[4 * j + 3] += q.w;
                                }
                            } else {
                                add_words(v, reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.residual) + at),
                                          p.aux_type);
                            }
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (col + j < p.n) v[j] += load_elem(p.residual, at + j, p.aux_type);
                        }
                    }
                    uint8_t* b = next_box(p.out_type == kF32);
                    if (p.out_type == kF32) {
                        put_f32(b, v);
                    } else {
                        uint32_t w[16];
                        pack32(v, w, p.out_type);
                        put_words(b, w);
                    }
                    if (p.out_tma)
                        send(b, map_out, col, out_row0, p.accumulate != 0);
                    else
                        copy_out(b, p.out, p.ldo, p.out_type == kF32 ? 4 : 2, row0, col);
                });
            } else if constexpr (EPI == kEpiSoftmax) {
                // Running maximum (of the scaled logits, base 2) and sum of
                // 2^(logit - maximum) of this row over this warp's columns,
                // the label's column left out.
                float top = -INFINITY, sum = 0.0f;
                const int32_t label = live ? load_label(p.labels, p.labels_i64, row, p.classes) : -1;
                const uint64_t scale = pair_f32(p.scale2, p.scale2);
                // Two chunks of a tile, from column col and col + kStep on. The
                // special-function units set the pace (a polynomial on the FMA
                // units for three eighths of the exponentials was slower, 707 us
                // instead of 621: the issue slots are needed too), so the rest
                // is two values an instruction.
                auto soft = [&](float* v, uint32_t col) {
                    const int32_t at = label - static_cast<int32_t>(col);
                    constexpr int kNext = static_cast<int>(kStep);
                    if ((at >= 0 && at < 32) || (at >= kNext && at < kNext + 32)) {
                        const int32_t place = at < 32 ? at : at - kNext + 32;
                        float z = 0.0f;
#pragma unroll
                        for (int j = 0; j < 64; ++j) {
                            z = j == place ? v[j] : z;
                            v[j] = j == place ? -INFINITY : v[j];  // its term is added by the join
                        }
                        p.label_dot[row] = z;
                    }
                    if (col + kStep + 32 > p.n) {  // past the last column: no weight
#pragma unroll
                        for (int j = 0; j < 64; ++j)
                            if (col + (j < 32 ? j : kStep - 32 + j) >= p.n) v[j] = -INFINITY;
                    }
                    float big[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                    for (int j = 4; j < 60; j += 8)
#pragma unroll
                        for (int h = 0; h < 4; ++h) big[h] = max3(big[h], v[j + 2 * h], v[j + 2 * h + 1]);
#pragma unroll
                    for (int h = 0; h < 4; ++h) big[h] = fmaxf(big[h], v[60 + h]);
                    const float most = fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3]));
                    const float now = fmaxf(top, most * p.scale2);
                    // A row whose logits so far are all -inf has no sum yet.
                    const float base = now == -INFINITY ? 0.0f : now;
                    const uint64_t minus = pair_f32(-base, -base);
                    uint64_t part[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 64; j += 2) {
                        const uint64_t x = fma2(pair_f32(v[j], v[j + 1]), scale, minus);
                        const float2 f = unpair_f32(x);
                        const uint64_t e = pair_f32(exp2_approx(f.x), exp2_approx(f.y));
                        part[(j >> 1) & 3] = add2(part[(j >> 1) & 3], e);
                    }
                    const float2 s2 = unpair_f32(add2(add2(part[0], part[1]), add2(part[2], part[3])));
                    sum = fmaf(sum, exp2_approx(top - base), s2.x + s2.y);
                    top = now;
                };
                // Tiles here are whole (128 * CG columns): batches of two chunks a warp.
                if constexpr (LONG) {
                    for (uint32_t tn = t.n0; ok && tn < t.n1; ++tn) {
                        float sums[32 * kMaxChunks];
                        ok = sum_pieces(t.p1 - t.p0, sums);
                        if (!ok) break;
#pragma unroll
                        for (int i = 0; i < kMaxChunks; i += 2) soft(sums + 32 * i, tn * bn_tile + group * 32 + i * kStep);
                    }
                } else {
                    for (uint32_t tn = t.n0; ok && tn < t.n1; ++tn) {
                        if (kSets == 2 && (acc & 1u) != set) {
                            ++acc;
                            continue;
                        }
                        uint32_t buf;
                        ok = wait_acc(buf);
                        if (!ok) break;
#pragma unroll 1
                        for (int i = 0; i < kMaxChunks; i += 2) {
                            float v[64];
                            issue(buf, i, v);
                            issue(buf, i + 1, v + 32);
                            arrived(v);
                            tie32(reinterpret_cast<int32_t*>(v + 32));
                            if (i + 2 == kMaxChunks) release(buf);
                            soft(v, tn * bn_tile + group * 32 + i * kStep);
                        }
                    }
                }
                if (ok && live) p.part[uint64_t(EW / 4 * t.segment + (e >> 2)) * p.m + row] = make_float2(top, sum);
            } else {
                const float lse2 = live ? p.lse2[row] : 0.0f;
                const float cmax_inv = largest > 0.0f ? 1.0f / largest : 0.0f;
                const float coef = live ? p.coef[row] * cmax_inv * p.grad_scale : 0.0f;
                // Column of the row's class here; negative where it has none or an earlier piece holds it.
                int32_t label = live ? load_label(p.labels, p.labels_i64, row, p.classes) : -1;
                if (label >= 0) label -= static_cast<int32_t>(p.class0);
                const uint32_t col_base = t.n0 * bn_tile + group * 32;
                const uint64_t scale = pair_f32(p.scale2, p.scale2), minus = pair_f32(-lse2, -lse2);
                const uint64_t weight = pair_f32(coef, coef);
                // Planes are read in whole K blocks of 64 columns.
                const uint32_t width = p.grad_planes == 1 ? p.n : (p.n + 63) / 64 * 64;
                ok = for_tile(t.p1 - t.p0, [&](float* v, int i) {
                    const uint32_t col = col_base + i * kStep;
                    if (row0 >= p.m || col >= width) return;
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 x = unpair_f32(fma2(pair_f32(v[j], v[j + 1]), scale, minus));
                        const float2 g = unpair_f32(mul2(pair_f32(exp2_approx(x.x), exp2_approx(x.y)), weight));
                        v[j] = g.x;
                        v[j + 1] = g.y;
                    }
                    const int32_t at = label - static_cast<int32_t>(col);
                    if (at >= 0 && at < 32) {
                        float g = 0.0f;
#pragma unroll
                        for (int j = 0; j < 32; ++j) {
                            if (j == at) g = v[j] -= coef;
                        }
                        if (p.grad_planes == 1 && col + at < p.n) {
                            const uint32_t w = pack2(g, 0.0f, p.in_type);
                            p.label_rest[row] = g - unpack2(w, p.in_type).x;
                        }
                    }
                    if (col + 32 > p.n) {  // pad columns hold zeros
#pragma unroll
                        for (int j = 0; j < 32; ++j)
                            if (col + j >= p.n) v[j] = 0.0f;
                    }
                    uint32_t w[16];
                    pack32(v, w, p.in_type);
                    uint8_t* b = next_box();
                    put_words(b, w);
                    send(b, map_out, col, row0, false);
                    if (p.grad_planes == 3) {
#pragma unroll
                        for (int plane = 1; plane < 3; ++plane) {
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                const float2 f = unpack2(w[j], kBF16);
                                v[2 * j] -= f.x;
                                v[2 * j + 1] -= f.y;
                            }
                            pack32(v, w, kBF16);
                            b = next_box();
                            put_words(b, w);
                            send(b, map_out, plane * p.grad_pitch + col, row0, false);
                        }
                    }
                });
            }
        }
        if (!ok && lane == 0) abort_all();
        if (lane == 0) bulk_wait_all();
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pk_issue_regs(EW)));
    }

    tc_fence_before();
    if constexpr (CG == 2)
        cluster_sync_all();
    else
        __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        if constexpr (CG == 2)
            tmem_dealloc_pair(tmem_base, kTmemCols);
        else
            tmem_dealloc(tmem_base, kTmemCols);
    }
}

}  // namespace knng_b200
