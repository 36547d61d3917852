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
// residual's type).  All sums and products are fp32.
#include "moe_kernels.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace moe {

// VEC values of one type, loaded and stored with 16-byte accesses (VEC 8) or
// one by one (VEC 1).
__device__ __forceinline__ void norm_load(const float *p, float (&v)[1]) { v[0] = *p; }
__device__ __forceinline__ void norm_load(const __nv_bfloat16 *p, float (&v)[1]) { v[0] = __bfloat162float(*p); }
__device__ __forceinline__ void norm_load(const __half *p, float (&v)[1]) { v[0] = __half2float(*p); }
__device__ __forceinline__ void norm_load(const float *p, float (&v)[8]) {
    const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void norm_load(const __nv_bfloat16 *p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void norm_load(const __half *p, float (&v)[8]) {
    const uint4 a = *reinterpret_cast<const uint4 *>(p);
    const uint32_t u[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void norm_store(float *p, const float (&v)[1]) { *p = v[0]; }
__device__ __forceinline__ void norm_store(__nv_bfloat16 *p, const float (&v)[1]) { *p = __float2bfloat16(v[0]); }
__device__ __forceinline__ void norm_store(__half *p, const float (&v)[1]) { *p = __float2half(v[0]); }
__device__ __forceinline__ void norm_store(float *p, const float (&v)[8]) {
    reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void norm_store(__nv_bfloat16 *p, const float (&v)[8]) {
    uint4 a;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    a.x = u[0]; a.y = u[1]; a.z = u[2]; a.w = u[3];
    *reinterpret_cast<uint4 *>(p) = a;
}
__device__ __forceinline__ void norm_store(__half *p, const float (&v)[8]) {
    uint4 a;
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 b = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        u[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    a.x = u[0]; a.y = u[1]; a.z = u[2]; a.w = u[3];
    *reinterpret_cast<uint4 *>(p) = a;
}

// The CTA's sum of v; `part` [33] is used by this call alone.  Warp totals are
// added in warp order by every thread, so the result does not depend on timing.
__device__ __forceinline__ float norm_cta_sum(float v, float *part) {
    v = warp_sum(v);
    const int nw = blockDim.x >> 5;
    if (nw == 1) return v;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (int)(threadIdx.x & 31) < nw ? part[threadIdx.x & 31] : 0.0f;
    return warp_sum(v);
}

// One CTA per row; thread i holds the chunks of VEC values at VEC * (i + c *
// blockDim.x), c < V.  SRC 0: y rows of type TY; 1: the combine of fp32 rows.
// Everything the row needs is loaded before the first sum, so that one memory
// latency covers it.
template <typename TR, typename TY, int VEC, int V, int SRC>
__global__ void __launch_bounds__(1024) k_block_norm(NormArgs a) {
    __shared__ float part[2][32];
    const int t = blockIdx.x;
    const int H = a.n_embd;
    const float inv_h = 1.0f / (float)H;   // each square is scaled first: the sum overflows only where the mean does
    float y[V][VEC], r[V][VEC], g[V][VEC], po[V][VEC];
    const TR *rr = (const TR *)a.r + (int64_t)t * a.ld_r;
    float gt[1] = {0.0f};
    if (a.gate_kind == NORM_GATE_TOKEN) norm_load((const TY *)a.gate + (int64_t)t * a.ld_gate, gt);
#pragma unroll
    for (int c = 0; c < V; ++c) {
        const int h = VEC * ((int)threadIdx.x + c * (int)blockDim.x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] = r[c][i] = po[c][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) g[c][i] = 0.0f;
        if (h >= H) continue;
        norm_load(rr + h, r[c]);
        if (SRC == 0 && a.y) norm_load((const TY *)a.y + (int64_t)t * a.ld_y + h, y[c]);
        if (a.gate_kind == NORM_GATE_FULL) norm_load((const TY *)a.gate + (int64_t)t * a.ld_gate + h, g[c]);
        else if (a.gate_kind == NORM_GATE_CHANNEL) norm_load((const float *)a.gate + h, g[c]);
        if (a.post) norm_load(a.post + h, po[c]);
    }
    if (SRC == 1) {
        // the chain of k_combine: fma from 0 in rank order, then + add.  Four
        // rows are in flight at a time.
        const float *rows = (const float *)a.y;
        const int32_t *pos = a.pos + (int64_t)t * a.k;
        const float *w = a.w + (int64_t)t * a.k;
        constexpr int U = VEC * V <= 8 ? 4 : 2;
        for (int j0 = 0; j0 < a.k; j0 += U) {
            float v[U][V][VEC], wj[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int at = j0 + u < a.k ? pos[j0 + u] : -1;
                wj[u] = j0 + u < a.k ? w[j0 + u] : 0.0f;
#pragma unroll
                for (int c = 0; c < V; ++c) {
                    const int h = VEC * ((int)threadIdx.x + c * (int)blockDim.x);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[u][c][i] = 0.0f;
                    if (h < H && at >= 0 && at < a.n_rows) norm_load(rows + (int64_t)at * a.ld_y + h, v[u][c]);
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
        if (a.add) {
#pragma unroll
            for (int c = 0; c < V; ++c) {
                const int h = VEC * ((int)threadIdx.x + c * (int)blockDim.x);
                if (h < H) {
                    float v[VEC];
                    norm_load(a.add + (int64_t)t * H + h, v);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) y[c][i] = __fadd_rn(y[c][i], v[i]);
                }
            }
        }
    }
    if (a.post) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < V; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) ss = fmaf(y[c][i] * inv_h, y[c][i], ss);
        const float inv = 1.0f / sqrtf(norm_cta_sum(ss, part[0]) + a.eps);
#pragma unroll
        for (int c = 0; c < V; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) y[c][i] *= inv * (po[c][i] + a.offset);
    }
    if (a.gate_kind != NORM_GATE_NONE) {
#pragma unroll
        for (int c = 0; c < V; ++c)
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float v = a.gate_kind == NORM_GATE_TOKEN ? gt[0] : g[c][i];
                y[c][i] *= a.sigmoid ? 1.0f / (1.0f + expf(-v)) : v;
            }
    }
    float ss = 0.0f;
    TR *ro = (TR *)a.r_out + (int64_t)t * a.ld_ro;
#pragma unroll
    for (int c = 0; c < V; ++c) {
        const int h = VEC * ((int)threadIdx.x + c * (int)blockDim.x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) r[c][i] = h < H ? fmaf(a.scale, y[c][i], r[c][i]) : 0.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) ss = fmaf(r[c][i] * inv_h, r[c][i], ss);
        if (h < H && a.r_out) norm_store(ro + h, r[c]);
        if (h < H && a.x && a.pre) norm_load(a.pre + h, po[c]);
    }
    if (!a.x) return;
    const float inv = 1.0f / sqrtf(norm_cta_sum(ss, part[1]) + a.eps);
    TY *xo = (TY *)a.x + (int64_t)t * a.ld_x;
#pragma unroll
    for (int c = 0; c < V; ++c) {
        const int h = VEC * ((int)threadIdx.x + c * (int)blockDim.x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) r[c][i] *= inv * (a.pre ? po[c][i] + a.offset : 1.0f);
        if (h < H) norm_store(xo + h, r[c]);
    }
}

template <typename TR, typename TY, int VEC, int SRC>
static cudaError_t norm_go(const NormArgs &a, cudaStream_t s) {
    const int chunks = (a.n_embd + VEC - 1) / VEC;
    // 8 values per thread where a CTA holds the row that way, else 16
    constexpr int V8 = 8 / VEC;
    const bool wide = chunks > 1024 * V8;
    const int per = wide ? 2 * V8 : V8;
    const int threads = ((chunks + per - 1) / per + 31) / 32 * 32;
    if (wide) k_block_norm<TR, TY, VEC, 2 * V8, SRC><<<a.n_tok, threads, 0, s>>>(a);
    else k_block_norm<TR, TY, VEC, V8, SRC><<<a.n_tok, threads, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename TR, typename TY>
static cudaError_t norm_types(const NormArgs &a, cudaStream_t s) {
    // 16-byte accesses need 8 values per chunk and aligned rows
    auto al = [](const void *p, int64_t ld, size_t size) {
        return !p || (((uintptr_t)p | (uintptr_t)(ld * (int64_t)size)) & 15) == 0;
    };
    const bool vec = a.n_embd % 8 == 0 && al(a.r, a.ld_r, sizeof(TR)) && al(a.r_out, a.ld_ro, sizeof(TR)) &&
                     al(a.y, a.ld_y, sizeof(TY)) && al(a.x, a.ld_x, sizeof(TY)) && al(a.add, a.n_embd, 4) &&
                     al(a.post, 0, 4) && al(a.pre, 0, 4) &&
                     (a.gate_kind == NORM_GATE_NONE || a.gate_kind == NORM_GATE_TOKEN ||
                      al(a.gate, a.gate_kind == NORM_GATE_FULL ? a.ld_gate : 0, sizeof(TY)));
    if (a.pos) {   // the expert rows of a layer are fp32
        if constexpr (std::is_same<TR, float>::value && std::is_same<TY, float>::value)
            return vec ? norm_go<TR, TY, 8, 1>(a, s) : norm_go<TR, TY, 1, 1>(a, s);
        else
            return cudaErrorInvalidValue;
    }
    return vec ? norm_go<TR, TY, 8, 0>(a, s) : norm_go<TR, TY, 1, 0>(a, s);
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
