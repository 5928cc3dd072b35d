// skinny.cuh -- x w^T for few rows of x (16 to a block), with the linear
// epilogue or the softmax pieces of product.cuh's kernel.
//
// Such a call reads w once and does little else, so it is bound by HBM on a
// large w and by latency on a small one. There is no staging and no pipeline
// to fill: every warp takes 16 rows of w straight from memory into the
// registers of mma.sync (w as the 16-row operand, 8 rows of x as columns),
// 32 bytes of each of two rows per thread and step: four threads read a whole
// 128-byte line of a row. Both operands use the same order of K inside a step,
// so a thread's 32 bytes are its fragments of four MMAs as they lie. Rows that are not 16-byte aligned are
// read element by element; no row is copied first. With few rows of w, up to
// eight warps share a row group and cut K between them. Arithmetic is a
// fraction of what mma.sync offers; the tensor memory would only add latency.
//
// Sums leave the tensor cores every 32 of K and are added to nearest in
// registers. One bf16 row against 100,000 x 960: 34 us, 5.6 TB/s; one fp32 row:
// 60.5 us, 6.3 TB/s; one bf16 row against 1024 x 960: 3.7 us.
//
// fp32 operands are multiplied by the fp32 units: at 4 bytes a value
// of w they keep up with HBM for 16 rows of x. The loads are the same; a
// thread's sums over its share of K are added over the four threads of a row.
#pragma once
#include "product.cuh"

namespace knng_b200 {

constexpr int kSkinnyRows = 16;         // rows of x a block takes
constexpr uint32_t kSkinnySmem = 96 * 1024;  // most shared memory for x

struct SkinnyParams {
    const void* x;
    const void* w;
    uint64_t ldx, ldw;
    uint32_t m, n, k;
    uint32_t pitch;        // bytes of a row of x in shared memory
    uint32_t ksplit;       // warps of a block that share a group of 16 rows: 1, 2, 4, 8
    int x_vec, w_vec;      // rows allow 16-byte loads (1), those of w perhaps 32-byte ones (2)
    // store
    const void* bias;
    const void* residual;
    uint64_t ldr;
    void* out;
    uint64_t ldo;
    int out_type;
    void* pre;
    uint64_t ldp;
    int activation;
    // softmax
    float scale2;
    const void* labels;
    int labels_i64;
    float2* part;          // [gridDim.x][m]
    float* label_dot;
};

// Columns of a step: 128 bytes of a row, 32 per thread.
__host__ __device__ constexpr uint32_t skinny_step(bool f32) { return f32 ? 32u : 64u; }

// Bytes of a row of x in shared memory: whole steps, and for the 16-bit
// fragments 16 more, so that eight rows meet no bank twice.
inline uint32_t skinny_pitch(uint32_t k, bool f32)
{
    return (k + skinny_step(f32) - 1) / skinny_step(f32) * 128 + (f32 ? 0 : 16);
}

__device__ __forceinline__ void mma_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1, bool bf16)
{
    if (bf16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// The 8 values at src[at] .. src[at + 7], of which `left` exist (the rest are
// zeros), as words: 4 of two 16-bit values, or 8 fp32.
template <int TYPE>
__device__ __forceinline__ void load8_words(const void* src, uint64_t at, uint32_t left, bool vec, uint32_t* out)
{
    if constexpr (TYPE == kF32) {
        const uint32_t* f = static_cast<const uint32_t*>(src) + at;
        if (vec && left >= 8) {
            const uint4 a = __ldcs(reinterpret_cast<const uint4*>(f)), b = __ldcs(reinterpret_cast<const uint4*>(f) + 1);
            out[0] = a.x, out[1] = a.y, out[2] = a.z, out[3] = a.w;
            out[4] = b.x, out[5] = b.y, out[6] = b.z, out[7] = b.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = j < static_cast<int>(left) ? f[j] : 0u;
        }
    } else {
        const uint16_t* h = static_cast<const uint16_t*>(src) + at;
        if (vec && left >= 8) {
            const uint4 q = __ldcs(reinterpret_cast<const uint4*>(h));
            out[0] = q.x, out[1] = q.y, out[2] = q.z, out[3] = q.w;
        } else {
            uint32_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = j < static_cast<int>(left) ? h[j] : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) out[j] = v[2 * j] | (v[2 * j + 1] << 16);
        }
    }
}

// A thread's 32 bytes of a row of w: columns c .. c + 7 of fp32, c .. c + 15 of
// 16 bits. One instruction where rows lie on 32-byte boundaries.
template <int TYPE>
__device__ __forceinline__ void load_w(const SkinnyParams& p, uint32_t row, uint32_t c, uint32_t* out)
{
    constexpr uint32_t kValues = TYPE == kF32 ? 8 : 16;
    const uint64_t at = row * p.ldw + c;
    const uint32_t left = row < p.n && c < p.k ? p.k - c : 0u;
    if (p.w_vec == 2 && left >= kValues) {
        asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(out[0]), "=r"(out[1]), "=r"(out[2]), "=r"(out[3]), "=r"(out[4]), "=r"(out[5]), "=r"(out[6]),
                       "=r"(out[7])
                     : "l"(static_cast<const uint8_t*>(p.w) + at * (TYPE == kF32 ? 4 : 2)));
    } else {
        load8_words<TYPE>(p.w, at, left, p.w_vec != 0, out);
        if constexpr (TYPE != kF32) load8_words<TYPE>(p.w, at + 8, left > 8 ? left - 8 : 0u, p.w_vec != 0, out + 4);
    }
}

// NT: tiles of 8 rows of x.
template <int TYPE, int NT, int EPI>
__global__ void __launch_bounds__(256) skinny_kernel(const SkinnyParams p)
{
    const uint32_t token0 = blockIdx.y * kSkinnyRows;
    const uint32_t tokens = min(p.m - token0, static_cast<uint32_t>(kSkinnyRows));
    constexpr int kWords = TYPE == kF32 ? 8 : 4;  // of 8 values
    extern __shared__ __align__(16) uint8_t xs[];
    __shared__ float red[8][NT * 4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;

    previous_done();

    // x into shared memory, 8 values a thread at a time, zeros past its rows
    // and columns.
    const uint32_t octets = p.pitch / (4 * kWords);
    for (uint32_t i = threadIdx.x; i < NT * 8 * octets; i += 256) {
        const uint32_t r = i / octets, c = (i - r * octets) * 8;
        uint32_t v[kWords];
        load8_words<TYPE>(p.x, (token0 + r) * p.ldx + c, r < tokens && c < p.k ? p.k - c : 0u, p.x_vec, v);
#pragma unroll
        for (int q = 0; q < kWords; q += 4)
            *reinterpret_cast<uint4*>(xs + r * p.pitch + c * (kWords / 2) + q * 4) =
                make_uint4(v[q], v[q + 1], v[q + 2], v[q + 3]);
    }
    __syncthreads();

    const uint32_t ks = warp % p.ksplit;
    const uint32_t per_block = 8 / p.ksplit;  // row groups of a block at a time
    const uint32_t groups = (p.n + 15) / 16;
    const uint32_t steps = (p.k + skinny_step(TYPE == kF32) - 1) / skinny_step(TYPE == kF32);
    // Rounds of the block: every warp takes part in the barriers of each.
    const uint32_t rounds = (groups + per_block - 1) / per_block;

    float top[2 * NT], sum[2 * NT];
    int32_t label[2 * NT];
    if constexpr (EPI == kEpiSoftmax) {
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
            const uint32_t token = (i >> 1) * 8 + 2 * t + (i & 1);
            top[i] = -INFINITY;
            sum[i] = 0.0f;
            label[i] = token < tokens ? load_label(p.labels, p.labels_i64, token0 + token, p.n) : -1;
        }
    }

    for (uint32_t rd = blockIdx.x; rd < rounds; rd += gridDim.x) {
        const uint32_t group = rd * per_block + warp / p.ksplit;
        const uint32_t r0 = group * 16 + g;
        // acc[q][0..3]: rows r0, r0, r0 + 8, r0 + 8 of w against rows 8 q + 2 t, + 1 of x.
        float acc[NT][4] = {};
        if constexpr (TYPE == kF32) {
            float f[2][NT * 8] = {};
            for (uint32_t s = ks; s < steps; s += 2 * p.ksplit) {
                uint32_t wa[2][8], wb[2][8];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t c = (s + u * p.ksplit) * 32 + t * 8;
                    load_w<TYPE>(p, r0, c, wa[u]);
                    load_w<TYPE>(p, r0 + 8, c, wb[u]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (s + u * p.ksplit >= steps) break;
#pragma unroll
                    for (int q = 0; q < NT * 8; ++q) {
                        if (q >= static_cast<int>(tokens)) break;
                        const float4* b = reinterpret_cast<const float4*>(xs + q * p.pitch + (s + u * p.ksplit) * 128 + t * 32);
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float4 v = b[h];
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const uint32_t* w = r ? wb[u] : wa[u];
                                f[r][q] = fmaf(__uint_as_float(w[4 * h]), v.x, f[r][q]);
                                f[r][q] = fmaf(__uint_as_float(w[4 * h + 1]), v.y, f[r][q]);
                                f[r][q] = fmaf(__uint_as_float(w[4 * h + 2]), v.z, f[r][q]);
                                f[r][q] = fmaf(__uint_as_float(w[4 * h + 3]), v.w, f[r][q]);
                            }
                        }
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < NT * 8; ++q) {
                if (q >= static_cast<int>(tokens)) break;
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float v = f[r][q];
                    v += __shfl_xor_sync(~0u, v, 1);
                    v += __shfl_xor_sync(~0u, v, 2);
                    if ((q & 7) >> 1 == t) acc[q >> 3][2 * r + (q & 1)] = v;
                }
            }
        } else {
            for (uint32_t s0 = ks; s0 < steps; s0 += 2 * p.ksplit) {
                uint32_t wa[2][8], wb[2][8];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t c = (s0 + u * p.ksplit) * 64 + t * 16;
                    load_w<TYPE>(p, r0, c, wa[u]);
                    load_w<TYPE>(p, r0 + 8, c, wb[u]);
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t s = s0 + u * p.ksplit;
                    if (s >= steps) break;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float part[NT][4] = {};
                        const uint32_t a0[4] = {wa[u][4 * h], wb[u][4 * h], wa[u][4 * h + 1], wb[u][4 * h + 1]};
                        const uint32_t a1[4] = {wa[u][4 * h + 2], wb[u][4 * h + 2], wa[u][4 * h + 3], wb[u][4 * h + 3]};
#pragma unroll
                        for (int q = 0; q < NT; ++q) {
                            const uint4 b =
                                *reinterpret_cast<const uint4*>(xs + (q * 8 + g) * p.pitch + s * 128 + t * 32 + h * 16);
                            mma_16816(part[q], a0, b.x, b.y, TYPE == kBF16);
                            mma_16816(part[q], a1, b.z, b.w, TYPE == kBF16);
                        }
#pragma unroll
                        for (int q = 0; q < NT; ++q)
#pragma unroll
                            for (int j = 0; j < 4; ++j) acc[q][j] += part[q][j];
                    }
                }
            }
        }
        if (p.ksplit > 1) {
#pragma unroll
            for (int q = 0; q < NT; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) red[warp][q * 4 + j][lane] = acc[q][j];
            __syncthreads();
            if (ks == 0) {
                for (uint32_t o = 1; o < p.ksplit; ++o)
#pragma unroll
                    for (int q = 0; q < NT; ++q)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[q][j] += red[warp + o][q * 4 + j][lane];
            }
            __syncthreads();
        }
        if (ks != 0) continue;
        if constexpr (EPI == kEpiStore) {
#pragma unroll
            for (int q = 0; q < NT; ++q)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t here = q * 8 + 2 * t + (j & 1);
                    const uint64_t token = token0 + here;
                    const uint32_t col = r0 + 8 * (j >> 1);
                    if (here >= tokens || col >= p.n) continue;
                    float z = acc[q][j];
                    if (p.bias) z += load_elem(p.bias, col, TYPE);
                    if (p.pre) store_elem(p.pre, token * p.ldp + col, z, TYPE);
                    z = act_dyn(z, p.activation);
                    if (p.residual) z += load_elem(p.residual, token * p.ldr + col, TYPE);
                    store_elem(p.out, token * p.ldo + col, z, p.out_type);
                }
        } else {
#pragma unroll
            for (int i = 0; i < 2 * NT; ++i) {
                float v[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t col = r0 + 8 * h;
                    v[h] = acc[i >> 1][2 * h + (i & 1)];
                    if (static_cast<int32_t>(col) == label[i]) {
                        p.label_dot[token0 + (i >> 1) * 8 + 2 * t + (i & 1)] = v[h];
                        v[h] = -INFINITY;  // its term is added by the join
                    }
                    if (col >= p.n) v[h] = -INFINITY;
                }
                const float now = fmaxf(top[i], fmaxf(v[0], v[1]) * p.scale2);
                const float base = now == -INFINITY ? 0.0f : now;
                sum[i] = sum[i] * exp2_approx(top[i] - base) + exp2_approx(fmaf(v[0], p.scale2, -base)) +
                         exp2_approx(fmaf(v[1], p.scale2, -base));
                top[i] = now;
            }
        }
    }

    if constexpr (EPI == kEpiSoftmax) {
        // Over the eight row lanes of the warp, then over the warps in order.
        __syncthreads();
        float2* parts = reinterpret_cast<float2*>(&red[0][0][0]);  // [8 warps][NT * 8]
#pragma unroll
        for (int i = 0; i < 2 * NT; ++i) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                const float t2 = __shfl_xor_sync(~0u, top[i], o), s2 = __shfl_xor_sync(~0u, sum[i], o);
                const float now = fmaxf(top[i], t2);
                const float base = now == -INFINITY ? 0.0f : now;
                sum[i] = sum[i] * exp2_approx(top[i] - base) + s2 * exp2_approx(t2 - base);
                top[i] = now;
            }
            if (g == 0) parts[warp * NT * 8 + (i >> 1) * 8 + 2 * t + (i & 1)] = make_float2(top[i], sum[i]);
        }
        __syncthreads();
        if (threadIdx.x < tokens) {
            float m0 = -INFINITY, s = 0.0f;
            for (int w = 0; w < 8; ++w) {
                const float2 q = parts[w * NT * 8 + threadIdx.x];
                const float now = fmaxf(m0, q.x);
                const float base = now == -INFINITY ? 0.0f : now;
                s = s * exp2_approx(m0 - base) + q.y * exp2_approx(q.x - base);
                m0 = now;
            }
            p.part[uint64_t(blockIdx.x) * p.m + token0 + threadIdx.x] = make_float2(m0, s);
        }
    }
}

}  // namespace knng_b200
