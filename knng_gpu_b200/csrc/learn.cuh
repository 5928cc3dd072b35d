// learn.cuh -- the kernels around the tensor-core product of product.cuh:
// staging of rows that TMA cannot read (odd strides, fp32), the joins of split
// products and of softmax pieces, dz = dy act'(pre) with its column sums. All
// are bound by HBM (one read, one write) or, on small calls, by launch latency.
#pragma once
#include "product.cuh"

namespace knng_b200 {

// Rows that become 16-bit operands.
struct StageJob {
    const void* x;
    uint64_t rows;
    uint32_t k;
    uint64_t ld;
    uint16_t* out;
    uint32_t pitch;       // columns of a plane of out, a multiple of 8
    const void* labels;   // where given, rows without a label become zeros
    int labels_i64;
    uint32_t classes;
    uint32_t blocks;      // of the launch that work on it (0: nothing to do)
};

// One plane copies 16-bit rows to a pitch that TMA can read, three split fp32
// values into bf16 parts x = h + m + l (each rounded to nearest from what is
// left; a finite value whose rounding would overflow is truncated). Columns
// past k are zeros. One thread per 8 columns.
template <int PLANES>
__device__ void stage_rows(const StageJob& p, uint32_t block)
{
    const uint32_t groups = p.pitch / 8;
    const uint64_t total = p.rows * groups;
    for (uint64_t i = block * uint64_t(256) + threadIdx.x; i < total; i += uint64_t(p.blocks) * 256) {
        const uint64_t r = i / groups;
        const uint32_t c0 = static_cast<uint32_t>(i - r * groups) * 8;
        const bool keep = !p.labels || load_label(p.labels, p.labels_i64, r, p.classes) >= 0;
        if constexpr (PLANES == 1) {
            const uint16_t* src = static_cast<const uint16_t*>(p.x) + r * p.ld;
            uint32_t w[4];
            if (keep && c0 + 8 <= p.k && (reinterpret_cast<uintptr_t>(src + c0) & 15) == 0) {
                const uint4 q = *reinterpret_cast<const uint4*>(src + c0);
                w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
            } else if (keep && c0 + 8 <= p.k && r > 0 && r + 1 < p.rows) {
                // Whole words, shifted by half a word where the row starts on
                // one; what they hold beside the eight values lies between the
                // first and the last row, so it is there to be read.
                const uintptr_t at = reinterpret_cast<uintptr_t>(src + c0);
                const uint32_t* word = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
                uint32_t v[5];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = word[j];
                const bool odd = at & 2;
                v[4] = odd ? word[4] : 0u;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = odd ? __funnelshift_r(v[j], v[j + 1], 16) : v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t a = keep && c0 + 2 * j < p.k ? src[c0 + 2 * j] : 0u;
                    const uint32_t b = keep && c0 + 2 * j + 1 < p.k ? src[c0 + 2 * j + 1] : 0u;
                    w[j] = a | (b << 16);
                }
            }
            *reinterpret_cast<uint4*>(p.out + r * p.pitch + c0) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
            const float* src = static_cast<const float*>(p.x) + r * p.ld;
            float v[8];
            if (keep && c0 + 8 <= p.k && (reinterpret_cast<uintptr_t>(src + c0) & 15) == 0) {
                const float4 a = *reinterpret_cast<const float4*>(src + c0);
                const float4 b = *reinterpret_cast<const float4*>(src + c0 + 4);
                v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
                v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = keep && c0 + j < p.k ? src[c0 + j] : 0.0f;
            }
            uint16_t* dst = p.out + r * (3ull * p.pitch) + c0;
#pragma unroll
            for (int plane = 0; plane < 3; ++plane) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t h2 = 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float& f = v[2 * j + h];
                        __nv_bfloat16 b = __float2bfloat16_rn(f);
                        if (isinf(__bfloat162float(b)) && !isinf(f)) b = __float2bfloat16_rz(f);
                        uint16_t bits;
                        memcpy(&bits, &b, 2);
                        h2 |= static_cast<uint32_t>(bits) << (16 * h);
                        f -= __bfloat162float(b);
                    }
                    w[j] = h2;
                }
                *reinterpret_cast<uint4*>(dst + uint64_t(plane) * p.pitch) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    }
}

struct JoinParams {
    const float* part;      // [splits][split_rows][pitch]
    uint32_t splits;
    uint64_t split_rows;
    uint32_t pitch;         // multiple of 4
    uint64_t m;
    uint32_t n;
    float alpha;
    const float* alpha_dev;  // the largest of alpha_parts values
    uint32_t alpha_parts;
    const void* bias;
    const void* residual;
    uint64_t ldr;
    int aux_type;
    int activation;
    void* out;
    uint64_t ldo;
    int out_type;
    void* pre;
    uint64_t ldp;
    const void* labels;     // rows without a label become zeros
    int labels_i64;
    uint32_t classes;
    const float* label_rest;  // with labels: row r also gets label_rest[r] * (row `label` of w), 16-bit rows
    const void* w;
    uint64_t ldw;
    int w_type;
    uint32_t blocks;        // of the launch that work on it (0: nothing to do)
};

// The pieces of a split product, summed in order, and the linear epilogue.
__device__ void join_splits(const JoinParams& p, uint32_t block)
{
    const uint32_t groups = (p.n + 3) / 4;
    const uint64_t total = p.m * groups;
    const float alpha = p.alpha_dev ? p.alpha * warp_largest(p.alpha_dev, p.alpha_parts) : p.alpha;
    for (uint64_t i = block * uint64_t(256) + threadIdx.x; i < total; i += uint64_t(p.blocks) * 256) {
        const uint64_t r = i / groups;
        const uint32_t c = static_cast<uint32_t>(i - r * groups) * 4;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        const int32_t label = p.labels ? load_label(p.labels, p.labels_i64, r, p.classes) : 0;
        if (label >= 0) {
            for (uint32_t s = 0; s < p.splits; ++s) {
                const float4 q = *reinterpret_cast<const float4*>(p.part + (s * p.split_rows + r) * p.pitch + c);
                v[0] += q.x, v[1] += q.y, v[2] += q.z, v[3] += q.w;
            }
            if (p.label_rest) {
                const float rest = p.label_rest[r];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (c + j < p.n) v[j] = fmaf(rest, load_elem(p.w, label * p.ldw + c + j, p.w_type), v[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= alpha;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (c + j >= p.n) break;
            float z = v[j];
            if (p.bias) z += load_elem(p.bias, c + j, p.aux_type);
            if (p.pre) store_elem(p.pre, r * p.ldp + c + j, z, p.aux_type);
            z = act_dyn(z, p.activation);
            if (p.residual) z += load_elem(p.residual, r * p.ldr + c + j, p.aux_type);
            store_elem(p.out, r * p.ldo + c + j, z, p.out_type);
        }
    }
}

// Joins a row's softmax pieces, which leave the label's own term out: with M
// the largest other score, S = sum of 2^(score - M) over the others and y the
// label's score, in base 2,
//   loss = log(1 + S 2^(M - y)), lse = y ln 2 + loss        where y >= M,
//   loss = (M - y) ln 2 + log(S + 2^(y - M)), lse likewise  where it is not.
// So the small loss of a well placed row keeps its digits. Without a label
// lse = M ln 2 + log S. LANES threads per row: a warp, or a block.
template <int LANES>
__global__ void __launch_bounds__(256) join_softmax_kernel(const float2* __restrict__ part, uint32_t pieces,
                                                           uint64_t m, const float* __restrict__ label_dot,
                                                           float scale2, const void* labels, int labels_i64,
                                                           uint32_t classes, float* __restrict__ loss,
                                                           float* __restrict__ lse)
{
    __shared__ float2 warps[8];
    previous_done();
    const uint64_t r = blockIdx.x * uint64_t(256 / LANES) + threadIdx.x / LANES;
    const int lane = threadIdx.x & 31;
    if (r >= m) return;
    float top = -INFINITY, sum = 0.0f;
    const auto merge = [&](float t2, float s2) {
        const float now = fmaxf(top, t2);
        const float base = now == -INFINITY ? 0.0f : now;
        sum = sum * exp2_approx(top - base) + s2 * exp2_approx(t2 - base);
        top = now;
    };
    for (uint32_t s = threadIdx.x % LANES; s < pieces; s += LANES) {
        const float2 q = part[uint64_t(s) * m + r];
        merge(q.x, q.y);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float t2 = __shfl_xor_sync(~0u, top, o), s2 = __shfl_xor_sync(~0u, sum, o);
        merge(t2, s2);
    }
    if constexpr (LANES > 32) {  // the row is the block's: no thread has left
        if (lane == 0) warps[threadIdx.x >> 5] = make_float2(top, sum);
        __syncthreads();
        if (threadIdx.x != 0) return;
        for (int w = 1; w < 8; ++w) merge(warps[w].x, warps[w].y);
    }
    if (lane == 0) {
        const bool has = load_label(labels, labels_i64, r, classes) >= 0;
        if (!has) {
            // No finite score: -inf, unless a NaN is among them.
            lse[r] = top == -INFINITY && sum == 0.0f ? top : fmaf(top, 0.69314718f, logf(sum));
            loss[r] = 0.0f;
        } else {
            const float y = label_dot[r] * scale2;
            if (!(y < top)) {  // also a NaN score
                const float others = sum == 0.0f ? y - y : log1pf(sum * exp2_approx(top - y));
                loss[r] = others;
                lse[r] = y == -INFINITY && sum == 0.0f ? y : fmaf(y, 0.69314718f, others);
            } else {
                const float tail = logf(sum + exp2_approx(y - top));
                loss[r] = fmaf(top - y, 0.69314718f, tail);
                lse[r] = fmaf(top, 0.69314718f, tail);
            }
        }
    }
}

// Per row of the gradient: coef = dloss scale and lse in base 2 (both 0 for a
// row without a label), and for each block of rows the largest finite |coef|.
struct GradRowsJob {
    const float* dloss;
    const float* lse;
    uint64_t m;
    float scale;
    const void* labels;
    int labels_i64;
    uint32_t classes;
    float* coef;
    float* lse2;
    float* largest;   // [blocks]
    uint32_t blocks;  // of the launch that work on it (0: nothing to do)
};

__device__ __forceinline__ void grad_rows(const GradRowsJob& p, uint32_t block)
{
    __shared__ float warps[8];
    float big = 0.0f;
    for (uint64_t r = block * uint64_t(256) + threadIdx.x; r < p.m; r += uint64_t(p.blocks) * 256) {
        const bool has = load_label(p.labels, p.labels_i64, r, p.classes) >= 0;
        const float c = has ? p.dloss[r] * p.scale : 0.0f;
        p.coef[r] = c;
        p.lse2[r] = has ? p.lse[r] * 1.44269504f : 0.0f;
        if (isfinite(c)) big = fmaxf(big, fabsf(c));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) big = fmaxf(big, __shfl_xor_sync(~0u, big, o));
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = big;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 8; ++w) big = fmaxf(big, warps[w]);
        p.largest[block] = big;
    }
}

// What comes before the products, in one launch: up to two matrices to stage,
// the rows of the gradient. Blocks are dealt out in that order. Bound by HBM:
// splitting 10,128 x 960 fp32 values takes 16 us for 97 MB, 6.0 TB/s.
struct PrepareParams {
    StageJob a, b;
    GradRowsJob rows;
};

template <int PLANES>
__global__ void __launch_bounds__(256) prepare_kernel(const PrepareParams p)
{
    previous_done();
    uint32_t block = blockIdx.x;
    if (block < p.a.blocks) {
        stage_rows<PLANES>(p.a, block);
    } else if ((block -= p.a.blocks) < p.b.blocks) {
        stage_rows<PLANES>(p.b, block);
    } else {
        grad_rows(p.rows, block - p.b.blocks);
    }
}

constexpr int kSlopeBlocks = 4;  // per SM, all resident

struct SlopeParams {
    const void* dy;
    uint64_t lddy;
    const void* pre;      // not read without an activation
    uint64_t ldp;
    uint64_t m;
    uint32_t n;
    uint16_t* out;        // dz as 16-bit operands (may be NULL: column sums only)
    uint32_t pitch;       // columns of a plane of out
    float* sums;          // [gy][n] column sums (may be NULL)
    int vec;              // rows of dy and pre allow 16-byte loads
    uint32_t gx, gy;      // blocks over columns and rows
    StageJob a, b;        // matrices that the products after it need staged
};

// 8 consecutive values as they lie; those past `left` are zeros.
template <int TYPE>
struct Octet {
    uint32_t w[TYPE == kF32 ? 8 : 4];

    __device__ __forceinline__ void load(const void* p, uint64_t at, uint32_t left, bool whole)
    {
        constexpr int kWords = TYPE == kF32 ? 8 : 4;
        if (whole) {
            const uint4* q = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + at * (kWords / 2));
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 v = __ldcs(q + i);
                w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
            }
        } else if constexpr (TYPE == kF32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = j < static_cast<int>(left) ? static_cast<const uint32_t*>(p)[at + j] : 0u;
        } else {
            const uint16_t* h = static_cast<const uint16_t*>(p) + at;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                w[j] = (2 * j < static_cast<int>(left) ? h[2 * j] : 0u) |
                       (2 * j + 1 < static_cast<int>(left) ? static_cast<uint32_t>(h[2 * j + 1]) << 16 : 0u);
        }
    }
    // Values 2 j and 2 j + 1.
    __device__ __forceinline__ uint64_t pair(int j) const
    {
        if constexpr (TYPE == kF32) return pair_f32(__uint_as_float(w[2 * j]), __uint_as_float(w[2 * j + 1]));
        const float2 f = unpack2(w[j], TYPE);
        return pair_f32(f.x, f.y);
    }
};

// dz = dy act'(pre), rounded to the operands' type, and its column sums (of
// the unrounded values). Bound by HBM: dy and pre in, dz out. A block takes 256
// columns (8 per lane) and a range of rows; its 8 warps take every eighth row,
// the loads of the next rows on their way while the current ones are worked
// on, and add up their sums in order. bf16 gelu, 100,000 x 1024: 111 us for 614
// MB, 5.5 TB/s.
template <int ACT, int TYPE>
__global__ void __launch_bounds__(256, kSlopeBlocks) slope_kernel(const SlopeParams p)
{
    constexpr int kRows = TYPE == kF32 ? 1 : 2;  // of a warp at a time
    constexpr int kOut = TYPE == kF16 ? kF16 : kBF16;
    constexpr int kPlanes = TYPE == kF32 ? 3 : 1;
    __shared__ float total[8][256];
    previous_done();
    if (blockIdx.x >= p.gx * p.gy) {
        const uint32_t block = blockIdx.x - p.gx * p.gy;
        if (block < p.a.blocks)
            stage_rows<kPlanes>(p.a, block);
        else
            stage_rows<kPlanes>(p.b, block - p.a.blocks);
        return;
    }
    const uint32_t bx = blockIdx.x % p.gx, by = blockIdx.x / p.gx;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t c0 = bx * 256 + lane * 8;
    const uint64_t r0 = p.m * by / p.gy, r1 = p.m * (by + 1) / p.gy;
    const uint32_t left = c0 < p.n ? p.n - c0 : 0;
    const bool whole = p.vec && left >= 8;
    uint64_t acc[4] = {0, 0, 0, 0};
    Octet<TYPE> dy[kRows], z[kRows];
    const auto fetch = [&](uint64_t r) {
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
            const bool there = left && r + 8 * h < r1;
            const uint64_t row = there ? r + 8 * h : 0;
            dy[h].load(p.dy, row * p.lddy + c0, there ? left : 0, there && whole);
            if constexpr (ACT != kActNone) z[h].load(p.pre, row * p.ldp + c0, there ? left : 0, there && whole);
        }
    };
    fetch(r0 + warp);
    for (uint64_t r = r0 + warp; r < r1; r += 8 * kRows) {
        Octet<TYPE> d[kRows], u[kRows];
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
            d[h] = dy[h];
            u[h] = z[h];
        }
        fetch(r + 8 * kRows);
#pragma unroll
        for (int h = 0; h < kRows; ++h) {
            if (r + 8 * h >= r1) break;
            float v[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint64_t g = d[h].pair(j);
                if constexpr (ACT != kActNone) g = mul2(g, slope2<ACT>(u[h].pair(j)));
                acc[j] = add2(acc[j], g);
                const float2 f = unpair_f32(g);
                v[2 * j] = f.x;
                v[2 * j + 1] = f.y;
            }
            if (p.out && c0 < p.pitch) {
                uint16_t* dst = p.out + (r + 8 * h) * (uint64_t(p.pitch) * kPlanes) + c0;
#pragma unroll
                for (int plane = 0; plane < kPlanes; ++plane) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[j] = pack2(v[2 * j], v[2 * j + 1], kOut);
                        if (plane + 1 < kPlanes) {
                            const float2 f = unpack2(w[j], kOut);
                            v[2 * j] -= f.x;
                            v[2 * j + 1] -= f.y;
                        }
                    }
                    *reinterpret_cast<uint4*>(dst + plane * p.pitch) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    }
    if (p.sums) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = unpair_f32(acc[j]);
            total[warp][lane * 8 + 2 * j] = f.x;
            total[warp][lane * 8 + 2 * j + 1] = f.y;
        }
        __syncthreads();
        const uint32_t c = bx * 256 + threadIdx.x;
        if (c < p.n) {
            float s = 0.0f;
            for (int w = 0; w < 8; ++w) s += total[w][threadIdx.x];
            p.sums[uint64_t(by) * p.n + c] = s;
        }
    }
}

// Column sums of [rows][n] partial sums: 32 columns per block, 8 row groups
// added in order.
struct SumsJob {
    const float* sums;
    uint32_t rows, n;
    void* out;
    int type;
    uint32_t blocks;  // of the launch that work on it (0: nothing to do)
};

__device__ __forceinline__ void join_sums(const SumsJob& p, uint32_t block)
{
    __shared__ float part[8][32];
    const int g = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t c = block * 32 + lane;
    float s = 0.0f;
    if (c < p.n)
        for (uint32_t r = g; r < p.rows; r += 8) s += p.sums[uint64_t(r) * p.n + c];
    part[g][lane] = s;
    __syncthreads();
    if (g == 0 && c < p.n) {
        float t = 0.0f;
        for (int i = 0; i < 8; ++i) t += part[i][lane];
        store_elem(p.out, c, t, p.type);
    }
}

// What comes after the products, in one launch: 4 to 7 us, mostly the latency
// of one pass over the pieces.
struct FinishParams {
    SumsJob sums;
    JoinParams a, b;
};

__global__ void __launch_bounds__(256) finish_kernel(const FinishParams p)
{
    previous_done();
    uint32_t block = blockIdx.x;
    if (block < p.sums.blocks) {
        join_sums(p.sums, block);
    } else if ((block -= p.sums.blocks) < p.a.blocks) {
        join_splits(p.a, block);
    } else {
        join_splits(p.b, block - p.a.blocks);
    }
}

}  // namespace knng_b200
