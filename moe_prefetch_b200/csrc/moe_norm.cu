// moe_norm.cu -- the norms around a block, with its gate and its residual:
//
//   y = the block's output row, or the combine sum_j w[t][j] rows[pos[t][j]]
//       (+ add[t]) of an expert layer
//   z = y * rsqrt(mean(y^2) + eps) * (post + offset)     (or y, without post)
//   r' = r + scale * act(gate) * z
//   x = r' * rsqrt(mean(r'^2) + eps) * (pre + offset)     (optional)
//
// One pass: y and r are read once, r' and x written once, and the row stays in
// registers over both norms (x is the norm of r' before its rounding to the
// residual's type).  All sums and products are fp32.  Bound by memory: 8,192 rows
// of 2,048 (bf16 beside an fp32 residual, a full gate) move 235 MB in 38.7 us, 6.1
// TB/s of a measured copy's 6.5; few rows are bound by latency (4 us for one row
// with the combine of eight).
#include "moe_kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace moe {

// VEC values of one type as they are in memory: one by one (VEC 1), two, four (16
// bytes of fp32, 8 of a 16-bit type) or eight of a 16-bit type.  A warp's
// access then covers neighbouring whole sectors.
template <typename T, int VEC> struct NormRaw;
template <typename T> struct NormRaw<T, 1> {
    T u;
    __device__ __forceinline__ void load(const T *p) { u = *p; }
    __device__ __forceinline__ void zero() { u = T(0.0f); }
    __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = (float)u; }
};
template <> struct NormRaw<float, 2> {
    float2 a;
    __device__ __forceinline__ void load(const float *p) { a = *reinterpret_cast<const float2 *>(p); }
    __device__ __forceinline__ void zero() { a = make_float2(0.0f, 0.0f); }
    __device__ __forceinline__ void get(float (&v)[2]) const { v[0] = a.x; v[1] = a.y; }
};
template <> struct NormRaw<float, 4> {
    float4 a;
    __device__ __forceinline__ void load(const float *p) { a = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void zero() { a = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void get(float (&v)[4]) const { v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; }
};
template <> struct NormRaw<float, 8> {   // the norm weights beside 16-bit rows
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = reinterpret_cast<const float4 *>(p)[0];
        b = reinterpret_cast<const float4 *>(p)[1];
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};
template <typename T, int VEC> struct NormRaw {   // 16 bits, VEC 2, 4 or 8
    uint32_t u[VEC / 2];
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (VEC == 8) {
            const uint4 a = *reinterpret_cast<const uint4 *>(p);
            u[0] = a.x; u[1] = a.y; u[2] = a.z; u[3] = a.w;
        } else if constexpr (VEC == 4) {
            const uint2 a = *reinterpret_cast<const uint2 *>(p);
            u[0] = a.x; u[1] = a.y;
        } else {
            u[0] = *reinterpret_cast<const uint32_t *>(p);
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) u[i] = 0;
    }
    __device__ __forceinline__ void get(float (&v)[VEC]) const {
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
            if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                v[2 * i] = __uint_as_float(u[i] << 16);
                v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
            } else {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            }
        }
    }
};
template <typename T, int VEC>
__device__ __forceinline__ void norm_load(const T *p, float (&v)[VEC]) {
    NormRaw<T, VEC> u;
    u.load(p);
    u.get(v);
}
__device__ __forceinline__ uint32_t norm_pack(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
__device__ __forceinline__ uint32_t norm_pack(float a, float b, __half) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T, int VEC>
__device__ __forceinline__ void norm_store(T *p, const float (&v)[VEC]) {
    if constexpr (VEC == 1) *p = T(v[0]);
    else if constexpr (VEC == 2 && std::is_same<T, float>::value) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
    else if constexpr (VEC == 2) *reinterpret_cast<uint32_t *>(p) = norm_pack(v[0], v[1], T());
    else if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    else if constexpr (VEC == 4)
        *reinterpret_cast<uint2 *>(p) = make_uint2(norm_pack(v[0], v[1], T()), norm_pack(v[2], v[3], T()));
    else
        *reinterpret_cast<uint4 *>(p) = make_uint4(norm_pack(v[0], v[1], T()), norm_pack(v[2], v[3], T()),
                                                   norm_pack(v[4], v[5], T()), norm_pack(v[6], v[7], T()));
}

// The CTA's sum of v; `part` [32] is this sum's alone until the CTA's next
// barrier.  Every thread adds the warps' totals in the same order, so the
// result does not depend on timing.
__device__ __forceinline__ float norm_cta_sum(float v, float *part) {
    v = warp_sum(v);
    const int nw = blockDim.x >> 5;
    if (nw == 1) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    if (nw <= 8) {   // (part past nw is zero: k_block_norm clears it)
        const float4 a = reinterpret_cast<const float4 *>(part)[0], b = reinterpret_cast<const float4 *>(part)[1];
        return ((a.x + a.y) + (a.z + a.w)) + ((b.x + b.y) + (b.z + b.w));
    }
    v = (int)(threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : 0.0f;
    return warp_sum(v);
}

// 1 / (1 + e^-v): expf and a reciprocal of one ulp (the argument is at least 1)
__device__ __forceinline__ float norm_sigmoid(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + expf(-v)));
    return r;
}

// B bytes (4, 8 or 16) into shared memory without a register.
template <int B>
__device__ __forceinline__ void norm_copy(void *dst, const void *src) {
    if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(dst)), "l"(src), "n"(B) : "memory");
}

// Bytes of a row in the ring: r, y, and the gate where it is full, each aligned to
// its chunks (n_embd is a multiple of VEC), the row to 16.
template <typename TR, typename TY>
__host__ __device__ __forceinline__ int norm_row_bytes(const NormArgs &a) {
    return (a.n_embd * (int)(sizeof(TR) + sizeof(TY) * (a.gate_kind == NORM_GATE_FULL ? 2 : 1)) + 15) & ~15;
}

// A CTA takes rows blockIdx.x, + gridDim.x, ...; thread i holds the chunks of VEC
// values at VEC * (i + c * blockDim.x), c < V.  SRC 0: y rows of type TY; 1: the
// combine of fp32 rows.  The norm weights stay in registers over the rows.  With
// S > 0, r, y and a full gate come through a ring of S rows in dynamic shared
// memory, each thread copying and reading its own chunks (so the ring needs no
// barrier): the kernel is bound by memory, and S - 1 rows are on their way while
// one is in its two sums.
// CTAs of 256 threads per SM: four, or three with more registers where that is
// faster (8,192 rows of 2,048, bf16 beside an fp32 residual with a full gate: 38.7
// us with three, 42.4 with four; all bf16, no gate: 27.0 and 29.1; 10,915 bf16 rows of
// 1,537: 84 and 131; fp32 rows of 1,000 are the other way: 45.8 with four, 50.9 with three).
template <typename TR, int VEC, int SRC, int THREADS, bool EXACT> constexpr int norm_ctas() {
    return THREADS > 256 ? 1 : SRC == 0 && (EXACT || VEC == 1 || sizeof(TR) == 2) ? 3 : 4;
}

template <typename TR, typename TY, int VEC, int V, int SRC, int THREADS, int S, bool EXACT>
__global__ void __launch_bounds__(THREADS, norm_ctas<TR, VEC, SRC, THREADS, EXACT>()) k_block_norm(NormArgs a) {
    static_assert(S == 0 || (SRC == 0 && VEC > 1), "the ring holds aligned rows");
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ __align__(16) float part[2][32];
    const int H = a.n_embd;
    const float inv_h = 1.0f / (float)H;   // each square is scaled first: the sum overflows only where the mean does
    auto at = [&](int c) { return VEC * ((int)threadIdx.x + c * (int)blockDim.x); };
    bool in_[V];
#pragma unroll
    for (int c = 0; c < V; ++c) in_[c] = at(c) < H;
    // whether the thread has chunk c: all of them (EXACT: 38.7 us of the case above, 44.5 without),
    // compared anew where registers are short, else kept
    auto in = [&](int c) {
        if constexpr (EXACT) return true;   // every thread has all its chunks
        else if constexpr (THREADS == 256 && VEC > 1) return at(c) < H;
        else return in_[c];
    };
    if (threadIdx.x < 64) (&part[0][0])[threadIdx.x] = 0.0f;
    if (threadIdx.x + 32 < 64 && blockDim.x == 32) (&part[0][0])[threadIdx.x + 32] = 0.0f;
    __syncthreads();
    pdl_enter();
    // the channel gate is folded into post in the kernels with a ring alone: without one that costs (777 rows
    // of 1,537 with a channel gate 8.9 -> 10.6 us)
    constexpr bool FOLD = S > 0;
    // the factors of y and of r', but for a full gate and the row's own: (post + offset) * act(channel gate),
    // and pre + offset; without FOLD the channel gate stays out of post
    float post[V][VEC], pre[V][VEC];
    auto load_weights = [&]() {
#pragma unroll
        for (int c = 0; c < V; ++c) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) post[c][i] = pre[c][i] = 0.0f;
            if (in(c) && a.post) norm_load(a.post + at(c), post[c]);
            if (in(c) && a.pre) norm_load(a.pre + at(c), pre[c]);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                post[c][i] = FOLD && !a.post ? 1.0f : post[c][i] + a.offset;
                pre[c][i] = a.pre ? pre[c][i] + a.offset : 1.0f;
            }
            if (FOLD && a.gate_kind == NORM_GATE_CHANNEL && in(c)) {
                float g[VEC];
                norm_load((const float *)a.gate + at(c), g);
#pragma unroll
                for (int i = 0; i < VEC; ++i) post[c][i] *= a.sigmoid ? norm_sigmoid(g[i]) : g[i];
            }
        }
    };
    NormRaw<TR, VEC> r_raw[V];
    NormRaw<TY, VEC> y_raw[V], g_raw[V];
#pragma unroll
    for (int c = 0; c < V; ++c) {   // what is not loaded below stays zero
        r_raw[c].zero();
        y_raw[c].zero();
        g_raw[c].zero();
    }
    float g_tok = 1.0f;
    auto load_row = [&](int64_t t) {
        const TY *gr = (const TY *)a.gate + t * a.ld_gate;   // (read where the gate is per token or full)
        if (a.gate_kind == NORM_GATE_TOKEN) {
            NormRaw<TY, 1> u;
            float v[1];
            u.load(gr);
            u.get(v);
            g_tok = v[0];
        }
#pragma unroll
        for (int c = 0; c < V; ++c) {
            if (!in(c)) continue;
            r_raw[c].load((const TR *)a.r + t * a.ld_r + at(c));
            if (SRC == 0 && a.y) y_raw[c].load((const TY *)a.y + t * a.ld_y + at(c));
            if (a.gate_kind == NORM_GATE_FULL) g_raw[c].load(gr + at(c));
        }
    };
    const int row_bytes = norm_row_bytes<TR, TY>(a);
    auto copy_row = [&](int64_t t, int stage) {
        uint8_t *dst = ring + stage * row_bytes;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int h = at(c);
            if (!in(c)) continue;
            norm_copy<VEC * (int)sizeof(TR)>(dst + h * (int)sizeof(TR), (const TR *)a.r + t * a.ld_r + h);
            uint8_t *dy = dst + H * (int)sizeof(TR) + h * (int)sizeof(TY);
            if (a.y) norm_copy<VEC * (int)sizeof(TY)>(dy, (const TY *)a.y + t * a.ld_y + h);
            if (a.gate_kind == NORM_GATE_FULL)
                norm_copy<VEC * (int)sizeof(TY)>(dy + H * (int)sizeof(TY), (const TY *)a.gate + t * a.ld_gate + h);
        }
    };
    auto read_row = [&](int64_t t, int stage) {
        const uint8_t *src = ring + stage * row_bytes;
        if (a.gate_kind == NORM_GATE_TOKEN) {
            float v[1];
            norm_load((const TY *)a.gate + t * a.ld_gate, v);
            g_tok = v[0];
        }
#pragma unroll
        for (int c = 0; c < V; ++c) {
            const int h = at(c);
            if (!in(c)) continue;
            r_raw[c].load((const TR *)src + h);
            const TY *sy = (const TY *)(src + H * (int)sizeof(TR)) + h;
            if (a.y) y_raw[c].load(sy);
            if (a.gate_kind == NORM_GATE_FULL) g_raw[c].load(sy + H);
        }
    };
    if (S) {
#pragma unroll
        for (int i = 0; i < S - 1; ++i) {
            if (blockIdx.x + (int64_t)i * gridDim.x < a.n_tok) copy_row(blockIdx.x + (int64_t)i * gridDim.x, i);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    }
    if (SRC == 0) load_weights();   // (behind the first rows' copies)
    int stage = 0;
    for (int64_t t = blockIdx.x; t < a.n_tok; t += gridDim.x) {
        if (S) {
            asm volatile("cp.async.wait_group %0;" ::"n"(S > 1 ? S - 2 : 0) : "memory");
            read_row(t, stage);
            const int64_t next = t + (int64_t)(S - 1) * gridDim.x;
            if (next < a.n_tok) copy_row(next, stage == 0 ? S - 1 : stage - 1);
            asm volatile("cp.async.commit_group;" ::: "memory");
            stage = stage + 1 == S ? 0 : stage + 1;
        } else {
            load_row(t);
        }
        float y[V][VEC], r[V][VEC], f[V][VEC];
        const float g_now = g_tok;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            r_raw[c].get(r[c]);
            y_raw[c].get(y[c]);
            g_raw[c].get(f[c]);
        }
        if (SRC == 1) {
            // the chain of k_combine: fma from 0 in rank order, then + add; U rows
            // are in flight at a time
            const float *rows = (const float *)a.y;
            const int32_t *pos = a.pos + t * a.k;
            const float *w = a.w + t * a.k;
            constexpr int U = THREADS == 256 && VEC > 1 ? 4 : 2;
            for (int j0 = 0; j0 < a.k; j0 += U) {
                float v[U][V][VEC], wj[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int q = j0 + u < a.k ? pos[j0 + u] : -1;
                    const bool have = q >= 0 && q < a.n_rows;
                    wj[u] = have ? w[j0 + u] : 0.0f;   // (an empty pair's weight may be anything)
#pragma unroll
                    for (int c = 0; c < V; ++c) {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) v[u][c][i] = 0.0f;
                        if (in(c) && have) norm_load(rows + (int64_t)q * a.ld_y + at(c), v[u][c]);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (j0 + u < a.k) {
#pragma unroll
                        for (int c = 0; c < V; ++c)
#pragma unroll
                            for (int i = 0; i < VEC; ++i) y[c][i] = __fmaf_rn(wj[u], v[u][c][i], y[c][i]);
                    }
            }
            load_weights();   // (one row per CTA: no earlier than they are needed)
            if (a.add) {
#pragma unroll
                for (int c = 0; c < V; ++c)
                    if (in(c)) {
                        float v[VEC];
                        norm_load(a.add + t * H + at(c), v);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) y[c][i] = __fadd_rn(y[c][i], v[i]);
                    }
            }
        }
        // the gate's factor (a token gate's not within by: the combine equals the norm of the combined rows bit
        // for bit, so every kernel multiplies in this order)
        if (a.gate_kind == NORM_GATE_TOKEN) {
            const float v = a.sigmoid ? norm_sigmoid(g_now) : g_now;
#pragma unroll
            for (int c = 0; c < V; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[c][i] = v;
        } else if (a.gate_kind == NORM_GATE_FULL || (!FOLD && a.gate_kind == NORM_GATE_CHANNEL)) {
#pragma unroll
            for (int c = 0; c < V; ++c) {
                if (!FOLD && a.gate_kind == NORM_GATE_CHANNEL && in(c)) norm_load((const float *)a.gate + at(c), f[c]);
                if (a.sigmoid) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) f[c][i] = norm_sigmoid(f[c][i]);
                }
            }
        }
        float by = a.scale;   // times scale, times post's 1 / sqrt
        if (a.post) {
            float ss = 0.0f;
#pragma unroll
            for (int c = 0; c < V; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) ss = fmaf(y[c][i] * inv_h, y[c][i], ss);
            by = a.scale * rsqrtf(norm_cta_sum(ss, part[0]) + a.eps);
        }
        if (!FOLD && !a.post) {
        } else if (a.gate_kind == NORM_GATE_NONE || (FOLD && a.gate_kind == NORM_GATE_CHANNEL)) {
#pragma unroll
            for (int c = 0; c < V; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[c][i] = post[c][i];
        } else {
#pragma unroll
            for (int c = 0; c < V; ++c)
#pragma unroll
                for (int i = 0; i < VEC; ++i) f[c][i] *= post[c][i];
        }
        float ss = 0.0f;
        TR *ro = (TR *)a.r_out + t * a.ld_ro;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            if (!in(c)) continue;       // (r is 0 there and adds nothing)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                // (without post and gate f is 1 where it is set at all: the same sum, of the same rounded product)
                r[c][i] = FOLD || a.post || a.gate_kind != NORM_GATE_NONE
                              ? fmaf(y[c][i] * by, f[c][i], r[c][i])
                              : __fadd_rn(__fmul_rn(by, y[c][i]), r[c][i]);
                ss = fmaf(r[c][i] * inv_h, r[c][i], ss);
            }
            if (a.r_out) norm_store(ro + at(c), r[c]);
        }
        if (!a.x) {
            __syncthreads();   // part[0] is read before the next row writes it
            continue;
        }
        const float inv = rsqrtf(norm_cta_sum(ss, part[1]) + a.eps);
        TY *xo = (TY *)a.x + t * a.ld_x;
#pragma unroll
        for (int c = 0; c < V; ++c) {
            if (!in(c)) continue;
#pragma unroll
            for (int i = 0; i < VEC; ++i) r[c][i] *= inv * pre[c][i];
            norm_store(xo + at(c), r[c]);
        }
        if (!a.post) __syncthreads();   // part[1] is read before the next row writes it
    }
}

// Rows wider than 8192, or wider than 2048 and of an odd width or alignment (VEC
// 1): a CTA per row keeps it in shared memory as fp32 (y, then r'), and each of
// the three passes has U chunks per thread in flight.  With a row in the registers
// of one CTA too few threads fit an SM: 2,046 rows of 8,200 in fp32 take 64 us
// (114 in registers), 3,928 of 4,271 in bf16 114 (206); 10,915 of 1,537 would take
// 110 (85).
template <typename TR, typename TY, int VEC, int SRC>
__global__ void __launch_bounds__(256) k_block_norm_wide(NormArgs a) {
    extern __shared__ __align__(16) float row[];   // [n_embd]
    __shared__ __align__(16) float part[2][32];
    constexpr int U = VEC == 1 ? 8 : VEC == 2 ? 4 : VEC == 4 ? 2 : 1;
    const int H = a.n_embd, step = VEC * (int)blockDim.x, h0 = VEC * (int)threadIdx.x;
    const float inv_h = 1.0f / (float)H;
    const int64_t t = blockIdx.x;
    if (threadIdx.x < 64) (&part[0][0])[threadIdx.x] = 0.0f;
    if (blockDim.x == 32) (&part[0][0])[threadIdx.x + 32] = 0.0f;
    __syncthreads();
    pdl_enter();
    const bool y_first = SRC == 1 || a.post;       // y is needed whole before r'
    float by = a.scale;
    if (y_first) {
        float ss = 0.0f;
        for (int b = h0; b < H; b += U * step) {
            float y[U][VEC];
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) y[u][i] = 0.0f;
                if (SRC == 0 && b + u * step < H) norm_load((const TY *)a.y + t * a.ld_y + b + u * step, y[u]);
            }
            if (SRC == 1) {   // the chain of k_combine: fma from 0 in rank order, then + add
                for (int j = 0; j < a.k; ++j) {
                    const int q = a.pos[t * a.k + j];
                    const bool have = q >= 0 && q < a.n_rows;
                    const float w = have ? a.w[t * a.k + j] : 0.0f;   // (an empty pair's weight may be anything)
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        float v[VEC];
#pragma unroll
                        for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
                        if (b + u * step < H && have)
                            norm_load((const float *)a.y + (int64_t)q * a.ld_y + b + u * step, v);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) y[u][i] = __fmaf_rn(w, v[i], y[u][i]);
                    }
                }
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (a.add && b + u * step < H) {
                        float v[VEC];
                        norm_load(a.add + t * H + b + u * step, v);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) y[u][i] = __fadd_rn(y[u][i], v[i]);
                    }
            }
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (b + u * step < H) {
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        row[b + u * step + i] = y[u][i];
                        ss = fmaf(y[u][i] * inv_h, y[u][i], ss);
                    }
                }
        }
        if (a.post) by *= rsqrtf(norm_cta_sum(ss, part[0]) + a.eps);
    }
    float g_tok = 1.0f;
    if (a.gate_kind == NORM_GATE_TOKEN) {
        float v[1];
        norm_load((const TY *)a.gate + t * a.ld_gate, v);
        g_tok = a.sigmoid ? norm_sigmoid(v[0]) : v[0];
    }
    const bool each = a.gate_kind == NORM_GATE_FULL || a.gate_kind == NORM_GATE_CHANNEL;
    float ss = 0.0f;
    for (int b = h0; b < H; b += U * step) {
        NormRaw<TR, VEC> r[U];
        NormRaw<TY, VEC> y[U], g[U];
        NormRaw<float, VEC> gc[U], po[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = b + u * step;
            if (h >= H) continue;
            r[u].load((const TR *)a.r + t * a.ld_r + h);
            if (!y_first && a.y) y[u].load((const TY *)a.y + t * a.ld_y + h);
            if (a.gate_kind == NORM_GATE_FULL) g[u].load((const TY *)a.gate + t * a.ld_gate + h);
            else if (each) gc[u].load((const float *)a.gate + h);
            if (a.post) po[u].load(a.post + h);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = b + u * step;
            if (h >= H) continue;
            float rv[VEC], yv[VEC], f[VEC], p[VEC];
            r[u].get(rv);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                f[i] = g_tok;
                p[i] = 1.0f - a.offset;
                yv[i] = y_first ? row[h + i] : 0.0f;
            }
            if (!y_first && a.y) y[u].get(yv);
            if (a.gate_kind == NORM_GATE_FULL) g[u].get(f);
            else if (each) gc[u].get(f);
            if (a.post) po[u].get(p);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                if (each && a.sigmoid) f[i] = norm_sigmoid(f[i]);
                if (a.post) f[i] *= p[i] + a.offset;
                rv[i] = fmaf(yv[i] * by, f[i], rv[i]);
                ss = fmaf(rv[i] * inv_h, rv[i], ss);
                row[h + i] = rv[i];
            }
            if (a.r_out) norm_store((TR *)a.r_out + t * a.ld_ro + h, rv);
        }
    }
    if (!a.x) return;
    const float inv = rsqrtf(norm_cta_sum(ss, part[1]) + a.eps);
    for (int b = h0; b < H; b += U * step) {
        NormRaw<float, VEC> pr[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (a.pre && b + u * step < H) pr[u].load(a.pre + b + u * step);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int h = b + u * step;
            if (h >= H) continue;
            float p[VEC], v[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) p[i] = 1.0f - a.offset;
            if (a.pre) pr[u].get(p);
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[i] = row[h + i] * (a.pre ? inv * (p[i] + a.offset) : inv);
            norm_store((TY *)a.x + t * a.ld_x + h, v);
        }
    }
}

template <typename TR, typename TY, int VEC, int V, int SRC, int THREADS, int S, bool EXACT = false>
static cudaError_t norm_launch(const NormArgs &a, int threads, cudaStream_t s) {
    // as many CTAs as the GPU holds, at most one per row; the combine takes a CTA
    // per row, since its own loads are many enough
    int dev = 0, sms = 0;
    cudaError_t e;
    if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
    if ((e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return e;
    int per_sm = (THREADS > 256 ? 1024 : 256 * norm_ctas<TR, VEC, SRC, THREADS, EXACT>()) / threads;
    const size_t smem = (size_t)S * norm_row_bytes<TR, TY>(a);
    if (S) {
        per_sm = std::min(per_sm, (int)(220 * 1024 / (smem + 2048)));
        static SmemAttr attr;
        if (smem > 40 * 1024 &&
            (e = attr.need((const void *)k_block_norm<TR, TY, VEC, V, SRC, THREADS, S, EXACT>, (int)smem)) != cudaSuccess)
            return e;
    }
    // 65,536 narrow rows: 24 CTAs of a warp for 16-bit rows (64 of bf16 24.5 us, with 16 CTAs 32.8 and 12
    // 30.5; beside fp32 r 31.7, 34.5, 38.8), 16 for fp32 (29.5; 24 CTAs 31.6)
    per_sm = std::min(sizeof(TY) == 2 ? 24 : 16, std::max(1, per_sm));
    return launch_pdl(k_block_norm<TR, TY, VEC, V, SRC, THREADS, S, EXACT>, SRC ? a.n_tok : std::min(a.n_tok, sms * per_sm), threads,
                      smem, s, 0, a);
}

template <typename TR, typename TY, int VEC, int SRC>
static cudaError_t norm_go(const NormArgs &a, cudaStream_t s) {
    const int chunks = (a.n_embd + VEC - 1) / VEC;
    if (a.n_embd > (VEC == 1 ? 2048 : 8192)) {
        const size_t smem = sizeof(float) * (size_t)a.n_embd;
        static SmemAttr attr;
        cudaError_t e;
        if (smem > 40 * 1024 && (e = attr.need((const void *)k_block_norm_wide<TR, TY, VEC, SRC>, (int)smem)) != cudaSuccess)
            return e;
        const int threads = std::min(256, (chunks + 255) / 256 * 32);   // eight chunks a thread while there are few
        return launch_pdl(k_block_norm_wide<TR, TY, VEC, SRC>, a.n_tok, threads, smem, s, 0, a);
    }
    constexpr int V = 8 / VEC;                      // 8 values per thread
    constexpr bool RING = VEC > 1 && SRC == 0;      // up to 12 bytes a value: 3 rows of 2048 (4 of 16 bits), 2 of 8192
    const int threads = ((chunks + V - 1) / V + 31) / 32 * 32;
    if constexpr (VEC > 1)
        if (threads > 256) return norm_launch<TR, TY, VEC, V, SRC, 1024, RING ? 2 : 0>(a, threads, s);
    constexpr int S = !RING ? 0 : sizeof(TR) == 2 ? 4 : 3;
    if constexpr (RING && VEC > 2)
        if (chunks == threads * V) return norm_launch<TR, TY, VEC, V, SRC, 256, S, true>(a, threads, s);
    return norm_launch<TR, TY, VEC, V, SRC, 256, S>(a, threads, s);
}

template <typename TR, typename TY>
static cudaError_t norm_types(const NormArgs &a, cudaStream_t s) {
    // chunks of VEC values: as wide as the width divides and every row is aligned to
    auto fits = [&](int vec) {
        auto al = [&](const void *p, int64_t ld, size_t size) {
            const uintptr_t m = std::min<uintptr_t>(16, vec * size) - 1;
            return !p || (((uintptr_t)p | (uintptr_t)(ld * (int64_t)size)) & m) == 0;
        };
        return a.n_embd % vec == 0 && al(a.r, a.ld_r, sizeof(TR)) && al(a.r_out, a.ld_ro, sizeof(TR)) &&
               al(a.y, a.ld_y, sizeof(TY)) && al(a.x, a.ld_x, sizeof(TY)) && al(a.add, a.n_embd, 4) && al(a.post, 0, 4) &&
               al(a.pre, 0, 4) &&
               (a.gate_kind == NORM_GATE_NONE || a.gate_kind == NORM_GATE_TOKEN ||
                (a.gate_kind == NORM_GATE_FULL ? al(a.gate, a.ld_gate, sizeof(TY)) : al(a.gate, 0, 4)));
    };
    constexpr int VEC = std::is_same<TR, float>::value ? 4 : 8;
    const int vec = fits(VEC) ? VEC : fits(2) ? 2 : 1;
    if (a.pos) {   // the expert rows of a layer are fp32
        if constexpr (std::is_same<TR, float>::value && std::is_same<TY, float>::value)
            return vec == VEC ? norm_go<TR, TY, VEC, 1>(a, s) : vec == 2 ? norm_go<TR, TY, 2, 1>(a, s) : norm_go<TR, TY, 1, 1>(a, s);
        else
            return cudaErrorInvalidValue;
    }
    return vec == VEC ? norm_go<TR, TY, VEC, 0>(a, s) : vec == 2 ? norm_go<TR, TY, 2, 0>(a, s) : norm_go<TR, TY, 1, 0>(a, s);
}

cudaError_t launch_block_norm(const NormArgs &a, int dt_r, int dt_y, cudaStream_t s) {
    if (a.n_tok == 0) return cudaSuccess;
    if (dt_r == DT_F32 && dt_y == DT_F32) return norm_types<float, float>(a, s);
    if (dt_r == DT_F32 && dt_y == DT_BF16) return norm_types<float, __nv_bfloat16>(a, s);
    if (dt_r == DT_F32 && dt_y == DT_F16) return norm_types<float, __half>(a, s);
    if (dt_r == DT_BF16 && dt_y == DT_BF16) return norm_types<__nv_bfloat16, __nv_bfloat16>(a, s);
    if (dt_r == DT_F16 && dt_y == DT_F16) return norm_types<__half, __half>(a, s);
    return cudaErrorInvalidValue;
}

}  // namespace moe
