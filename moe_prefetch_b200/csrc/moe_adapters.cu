// moe_adapters.cu -- low-rank adapters of many requests beside one projection:
//
//   out[t] = y[t] + scale[a] * B[a] (A[a] x[t]),   a = ids[t]
//
// with A [rank][n_in] and B [n_out][rank] in 16 bits.
//
// k_adapters: a cluster of CTAs takes one tile of up to M tokens that use the
// same adapter, wherever they stand in the batch (each CTA finds its tile's
// tokens from the ids itself, so there is no grouping launch and no
// workspace).  The cluster's CTAs split n_in for the first product, add their
// partial A x through distributed shared memory, and split n_out for the
// second.  The weights of an adapter are then read once per tile, x once, and
// y and out once.
//
// The work is bound by memory (2 * rank flops per 16-bit weight and row) and
// for few tokens by latency, so the products run on warp-level mma: a tcgen05
// tile has at least 64 rows and a TMEM round trip, and decoded tokens fill a
// few rows of one adapter.  16-bit x and all weights are exact operands.  An
// fp32 x is split into two tf32 parts, which leave out less than 2^-22 of it.  A x
// stays in fp32 until the second product, which splits it into parts of the
// weights' type, each rounded to the nearest: two for a 16-bit output (bf16:
// 2^-17 of a term is left out, against the output's own half step of 2^-8) and
// for fp16 weights (2^-23, each row scaled into fp16's range by a power of two),
// three bf16 parts (2^-26) for an fp32 output.
//
// Measured: 4,096 prompt tokens, 8 adapters of rank 64, 2048 -> 2048, all bf16: 28.6
// us (54 MB, 8.3 us of a measured copy; finding the tile 3.6 us, first product 7,
// the sums' exchange 5, second product 10; the tensor pipe is 24 % busy).  32
// requests, 16 adapters of rank 16, fp32: 7.8 us; one token, rank 8, 2048 -> 128:
// 5.6 us.
#include "moe_kernels.h"

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

namespace moe {

namespace {

constexpr int AD_THREADS = 256;
constexpr int AD_WARPS = AD_THREADS / 32;
constexpr int AD_IDS = 16;            // ids per thread and pass of the search

// columns of x per step of the first product: one k16 step per warp (M = 16), two per warp (M = 64)
template <int M> constexpr int ad_kc() { return M == 16 ? 128 : 64; }
// output columns per step of the second product: 2 (M = 16) or 4 (M = 64) mma tiles per warp
template <int M> constexpr int ad_nc() { return M == 16 ? 128 : 64; }

struct AdSmem {   // byte offsets in dynamic shared memory
    int x_stage, a_stage, stages;   // the ring of the first product: stages * (x_stage + a_stage)
    int b_stage, y_stage, b_stages, off_b;   // the ring of the second: b_stages * (b_stage + y_stage)
    // over the first ring once it is done: partial sums of the warps, then the
    // parts of A x (at 0); the CTA's partial A x (off_part)
    int off_part;
    int off_hist;                   // [n_adapters + 1]
    int bytes;
};

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, int bytes) {   // zero-fills to 16
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {   // tf32
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// v = hi + lo: hi is v rounded to the 11 bits of tf32 (from 2^127 on cut off to them, so
// that no finite v becomes infinite), lo the rest, at most 2^-11 of v, of which the
// mma reads 11 bits: the two are off by less than 2^-22 of v (2^-21 from 2^127 on).
// With hi cut off everywhere that was 2^-21; rounding lo as well gives 2^-23, and
// the router's adapters of 4,096 tokens in 19.4 us instead of 18.6.
__device__ __forceinline__ void split(float v, uint32_t &hi, uint32_t &lo) {
    hi = (__float_as_uint(v) + (fabsf(v) < 0x1p127f ? 0x1000u : 0u)) & 0xffffe000u;
    lo = v == __uint_as_float(hi) ? 0u : __float_as_uint(v - __uint_as_float(hi));   // (inf - inf is no remainder)
}

// two 16-bit weights as exact tf32 operands
__device__ __forceinline__ void pair32(uint32_t u, uint32_t &b0, uint32_t &b1, __nv_bfloat16) {
    b0 = u << 16;
    b1 = u & 0xffff0000u;
}
__device__ __forceinline__ void pair32(uint32_t u, uint32_t &b0, uint32_t &b1, __half) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&u));
    b0 = __float_as_uint(f.x);
    b1 = __float_as_uint(f.y);
}

__device__ __forceinline__ uint2 ad_pack(const float (&v)[4], __nv_bfloat16) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}
__device__ __forceinline__ uint2 ad_pack(const float (&v)[4], __half) {
    const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
    return make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
}

// two neighbouring outputs in shared memory: u += f * (v0, v1)
__device__ __forceinline__ void ad_add2(float *u, float v0, float v1, float f, bool fresh) {
    float2 y = make_float2(0.0f, 0.0f);
    if (!fresh) y = *reinterpret_cast<const float2 *>(u);
    *reinterpret_cast<float2 *>(u) = make_float2(fmaf(v0, f, y.x), fmaf(v1, f, y.y));
}
template <typename T>
__device__ __forceinline__ void ad_add2(T *u, float v0, float v1, float f, bool fresh) {
    uint32_t y0 = 0, y1 = 0;
    if (!fresh) pair32(*reinterpret_cast<const uint32_t *>(u), y0, y1, T());
    const float a = fmaf(v0, f, __uint_as_float(y0)), b = fmaf(v1, f, __uint_as_float(y1));
    if constexpr (std::is_same<T, __half>::value)
        *reinterpret_cast<__half2 *>(u) = __floats2half2_rn(a, b);
    else
        *reinterpret_cast<__nv_bfloat162 *>(u) = __floats2bfloat162_rn(a, b);
}

__device__ __forceinline__ void cp4(uint32_t dst, const void *src, int bytes) {   // zero-fills to 4
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// 16 bytes of an aligned row of n weights from i on; zeros from n on and for a
// null row
template <typename T>
__device__ __forceinline__ void row16(uint8_t *dst, const T *row, int i, int n) {
    const int have = row ? min(max(n - i, 0), 8) : 0;
    if (have) cp16(smem_u32(dst), row + i, 2 * have);
    else *reinterpret_cast<uint4 *>(dst) = make_uint4(0, 0, 0, 0);
}
// one element of a row at any alignment (fp32 asynchronously); zero for have = false
__device__ __forceinline__ void elem(uint8_t *dst, const float *src, bool have, const void *any) {
    cp4(smem_u32(dst), have ? (const void *)src : any, have ? 4 : 0);
}
template <typename T>
__device__ __forceinline__ void elem(uint8_t *dst, const T *src, bool have, const void *) {
    *reinterpret_cast<T *>(dst) = have ? *src : T(0.0f);
}

}  // namespace

// The tile of cluster `b`: its adapter (n_adapters: none) and tokens.  The
// tokens of an adapter keep their order and are cut into tiles of M.  False: no
// such tile.  Every CTA of a cluster finds the same.
template <int M>
__device__ __forceinline__ bool ad_find_tile(const AdapterArgs &p, int b, int *hist, int *s_tok, int &a_out, int &cnt_out) {
    __shared__ int s_wc[AD_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int na = p.n_adapters, n = p.n_tok, buckets = na + (p.y == p.out ? 0 : 1);   // in place, rows without an adapter stay
    const uint32_t below = (1u << lane) - 1;
    auto bucket = [&](int t) {   // -1: no token
        if (t >= n) return -1;
        const int v = __ldg(p.ids + t);
        return v >= 0 && v < na ? v : na;
    };
    if (n <= 32) {   // one token per lane, every warp alike: a tile is known by its first token
        const int id = bucket(lane);
        const uint32_t same = __match_any_sync(MOE_FULL, id);
        const int rank = __popc(same & below);
        const uint32_t heads = __ballot_sync(MOE_FULL, id >= 0 && id < buckets && rank % M == 0);
        const uint32_t me = __ballot_sync(MOE_FULL, (heads >> lane & 1) && __popc(heads & below) == b);
        if (!me) return false;
        const int l = __ffs(me) - 1;
        a_out = __shfl_sync(MOE_FULL, id, l);
        const int r0 = __shfl_sync(MOE_FULL, rank, l);
        cnt_out = min(M, __popc(__shfl_sync(MOE_FULL, same, l)) - r0);
        if (warp == 0) {
            if (id == a_out && rank >= r0 && rank < r0 + M) s_tok[rank - r0] = lane;
            if (lane >= cnt_out && lane < M) s_tok[lane] = -1;
        }
        static_assert(M <= 64, "the entries past a short tile are cleared below");
        if (M > 32 && warp == 1 && lane + 32 < M) s_tok[lane + 32] = -1;
        __syncthreads();
        return true;
    }
    // count the tokens of each adapter, then look for tile b.  A thread holds up
    // to AD_IDS neighbouring ids, whose runs it counts with one addition each.
    const int per = min(AD_IDS, (n + AD_THREADS - 1) / AD_THREADS), block = AD_THREADS * per;
    int id[AD_IDS];
    auto load = [&](int base) {
        const int t0 = base + tid * per;
        if (per == AD_IDS && ((uintptr_t)p.ids & 15) == 0 && base + block <= n) {
#pragma unroll
            for (int i = 0; i < AD_IDS; i += 4) {
                const int4 v = __ldg(reinterpret_cast<const int4 *>(p.ids + t0 + i));
                id[i] = v.x; id[i + 1] = v.y; id[i + 2] = v.z; id[i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < AD_IDS; ++i)
                if (i < per) id[i] = __ldg(p.ids + min(t0 + i, n - 1));
        }
#pragma unroll
        for (int i = 0; i < AD_IDS; ++i)
            id[i] = i >= per || t0 + i >= n ? -1 : id[i] >= 0 && id[i] < na ? id[i] : na;
    };
    load(0);
    for (int i = tid; i < na + 1; i += AD_THREADS) hist[i] = 0;
    if (tid < M) s_tok[tid] = -1;
    __syncthreads();
    for (int base = 0; base < n; base += block) {
        if (base) load(base);
        int run = 1;
#pragma unroll
        for (int i = 0; i < AD_IDS; ++i) {
            if (i >= per) break;
            const int next = i + 1 < AD_IDS ? id[i + 1 < AD_IDS ? i + 1 : i] : -1;
            if (i + 1 < per && next == id[i]) ++run;
            else {
                if (id[i] >= 0) atomicAdd(hist + id[i], run);
                run = 1;
            }
        }
    }
    __syncthreads();
    int a = -1, j0 = 0, before = 0;
    for (int i0 = 0; i0 < buckets && a < 0; i0 += 32) {   // every warp alike
        const int c = i0 + lane < buckets ? hist[i0 + lane] : 0;
        const int tiles = (c + M - 1) / M;
        int end = tiles;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(MOE_FULL, end, off);
            if (lane >= off) end += o;
        }
        const uint32_t in = __ballot_sync(MOE_FULL, b < before + end);
        if (in) {
            const int l = __ffs(in) - 1;
            a = i0 + l;
            j0 = (b - before - (__shfl_sync(MOE_FULL, end, l) - __shfl_sync(MOE_FULL, tiles, l))) * M;
            cnt_out = min(M, __shfl_sync(MOE_FULL, c, l) - j0);
        }
        before += __shfl_sync(MOE_FULL, end, 31);
    }
    if (a < 0) return false;
    a_out = a;
    // its tokens: those of rank [j0, j0 + M) among the adapter's
    int run = 0;
    for (int base = 0; base < n && run < j0 + M; base += block) {
        if (n > block) load(base);
        int mine = 0;
#pragma unroll
        for (int i = 0; i < AD_IDS; ++i) mine += id[i] == a ? 1 : 0;
        int pos = mine;   // inclusive prefix over the warp, then over the warps
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int o = __shfl_up_sync(MOE_FULL, pos, off);
            if (lane >= off) pos += o;
        }
        if (lane == 31) s_wc[warp] = pos;
        __syncthreads();
        pos += run - mine - j0;
#pragma unroll
        for (int w = 0; w < AD_WARPS; ++w) {
            const int c = s_wc[w];
            if (w < warp) pos += c;
            run += c;
        }
        if (mine && pos < M && pos + mine > 0) {
            const int t0 = base + tid * per;
#pragma unroll
            for (int i = 0; i < AD_IDS; ++i)
                if (id[i] == a) {
                    if (pos >= 0 && pos < M) s_tok[pos] = t0 + i;
                    ++pos;
                }
        }
        __syncthreads();
    }
    return true;
}

// out rows of the tile = y rows (or zeros), columns [o0, o1): rows without an
// adapter, or of an adapter of rank 0.
template <typename TO>
__device__ __forceinline__ void ad_copy_rows(const AdapterArgs &p, const int *s_tok, int cnt, int o0, int o1) {
    for (int m = threadIdx.x >> 5; m < cnt; m += AD_WARPS) {
        const int64_t t = s_tok[m];
        const TO *y = (const TO *)p.y + t * p.ld_y;
        TO *out = (TO *)p.out + t * p.ld_out;
        for (int o = o0 + (int)(threadIdx.x & 31); o < o1; o += 32) out[o] = p.y ? y[o] : TO(0.0f);
    }
}

// grid: tiles * cluster; M tokens per tile, up to 8 * NT ranks.  vec_x, vec_o: the
// rows of x, and of y and out, start at 16-byte boundaries.
template <typename TX, typename TW, typename TO, int M, int NT>
__global__ void __launch_bounds__(AD_THREADS, NT > 8 ? 1 : 2) k_adapters(AdapterArgs p, AdSmem L, int vec_x, int vec_o) {
    namespace cg = cooperative_groups;
    constexpr bool X16 = sizeof(TX) == 2;
    constexpr bool SCALED = std::is_same<TW, __half>::value;
    constexpr int P = !SCALED && sizeof(TO) == 4 ? 3 : 2;        // parts of A x
    constexpr int KC = ad_kc<M>(), NC = ad_nc<M>();
    constexpr int MT = M / 16, KW = AD_WARPS / MT;   // warps: MT row tiles x KW shares of the k steps
    constexpr int XP = KC * (int)sizeof(TX) + (X16 ? 16 : 32);   // row pitches in bytes, free of bank conflicts
    constexpr int AP = KC * 2 + 16;
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ int s_tok[M];
    __shared__ float s_fac[M];
    cg::cluster_group cl = cg::this_cluster();
    const int C = (int)cl.num_blocks(), cr = (int)cl.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int a, cnt;
    pdl_enter();
    if (!ad_find_tile<M>(p, blockIdx.x / C, reinterpret_cast<int *>(sm + L.off_hist), s_tok, a, cnt)) return;
    const int oc = (p.n_out + NC - 1) / NC;                  // output steps, this CTA's [s0, s1)
    const int s0 = (int)((int64_t)cr * oc / C), s1 = (int)((int64_t)(cr + 1) * oc / C);
    int rank = 0;
    if (a < p.n_adapters) rank = p.ranks ? min(max(p.ranks[a], 0), p.rank) : p.rank;
    if (rank == 0) {
        if (p.y != p.out) ad_copy_rows<TO>(p, s_tok, cnt, s0 * NC, min(s1 * NC, p.n_out));
        return;
    }
    const int r8 = (rank + 7) & ~7, nt = r8 / 8;     // ranks computed by the first product
    const int r16 = (rank + 15) & ~15;               // and read by the second: zeros from `rank` on
    const TW *A = (const TW *)p.a + (int64_t)a * p.rank * p.lda;
    const TW *B = (const TW *)p.b + (int64_t)a * p.n_out * p.rank;
    const int bp = ((p.rank + 15) & ~15) * 2 + 16;   // pitch of B and of the parts of A x

    // ---- loads: chunk k of x and A for the first product, chunk o of B and y for the second.
    // A whole chunk of aligned rows goes by 16 bytes, a thread always loading the same columns of the
    // same rows; others go by elements, neighbouring threads taking neighbouring elements.
    constexpr int XE = 16 / (int)sizeof(TX), XC = KC / XE, XR = AD_THREADS / XC, XN = M / XR;   // x: XN rows per thread
    constexpr int AC = KC / 8, AR = AD_THREADS / AC, AN = (8 * NT + AR - 1) / AR;
    static_assert(M % XR == 0, "whole passes over the rows of x");
    const TX *xrow[XN];
#pragma unroll
    for (int j = 0; j < XN; ++j) {
        const int t = s_tok[tid / XC + j * XR];
        xrow[j] = t >= 0 ? (const TX *)p.x + (int64_t)t * p.ld_x : nullptr;
    }
    const uint32_t sm0 = smem_u32(sm);
    auto load_k = [&](int k, int stage) {
        const int xo = stage * (L.x_stage + L.a_stage) + tid / XC * XP + 16 * (tid % XC);
        const int ao = stage * (L.x_stage + L.a_stage) + L.x_stage + tid / AC * AP + 16 * (tid % AC);
        const int xc = k * KC + XE * (tid % XC), ac = k * KC + 8 * (tid % AC);
        if (vec_x && (k + 1) * KC <= p.n_in) {
#pragma unroll
            for (int j = 0; j < XN; ++j)
                cp16(sm0 + xo + j * XR * XP, (xrow[j] ? xrow[j] : (const TX *)p.x) + xc, xrow[j] ? 16 : 0);
#pragma unroll
            for (int j = 0; j < AN; ++j) {
                const int r = tid / AC + j * AR;
                if (r < r8) cp16(sm0 + ao + j * AR * AP, A + (r < rank ? r * p.lda : 0) + ac, r < rank ? 16 : 0);
            }
            return;
        }
        for (int i = tid; i < M * KC; i += AD_THREADS) {
            const int t = s_tok[i / KC], col = k * KC + i % KC;
            elem(sm + stage * (L.x_stage + L.a_stage) + i / KC * XP + i % KC * (int)sizeof(TX),
                 (const TX *)p.x + (int64_t)max(t, 0) * p.ld_x + col, t >= 0 && col < p.n_in, p.x);
        }
#pragma unroll
        for (int j = 0; j < AN; ++j) {
            const int r = tid / AC + j * AR;
            if (r < r8) row16<TW>(sm + ao + j * AR * AP, r < rank ? A + (int64_t)r * p.lda : nullptr, ac, (int)p.lda);
        }
    };
    constexpr int BT = AD_THREADS / NC, BN = NT > BT ? NT / BT : 1;      // B: threads per row, 16-byte columns of each
    constexpr int YP = NC * (int)sizeof(TO) + (sizeof(TO) == 4 ? 32 : 16);
    constexpr int YE = 16 / (int)sizeof(TO), YC = NC / YE, YR = AD_THREADS / YC, YN = M / YR;   // y and out
    static_assert(M % YR == 0, "whole passes over the rows of y");
    int yt[YN];
#pragma unroll
    for (int j = 0; j < YN; ++j) yt[j] = s_tok[tid / YC + j * YR];
    auto load_b = [&](int o, int stage) {
        const int so = L.off_b + stage * (L.b_stage + L.y_stage);
        const int bo = so + tid / BT * bp + 16 * (tid % BT), yo = so + L.b_stage + tid / YC * YP + 16 * (tid % YC);
        const int row = o * NC + tid / BT, yc = o * NC + YE * (tid % YC);
        const bool full = (o + 1) * NC <= p.n_out;
#pragma unroll
        for (int j = 0; j < BN; ++j) {
            const int c = tid % BT + j * BT;
            if (8 * c >= r16) continue;
            const TW *src = B + (int64_t)row * p.rank;
            if (full && 8 * c + 8 <= rank) cp16(sm0 + bo + 16 * BT * j, src + 8 * c, 16);
            else row16<TW>(sm + bo + 16 * BT * j, row < p.n_out ? src : nullptr, 8 * c, rank);
        }
        if (!p.y) return;
        if (vec_o && full) {
#pragma unroll
            for (int j = 0; j < YN; ++j)
                if (yt[j] >= 0) cp16(sm0 + yo + j * YR * YP, (const TO *)p.y + (int64_t)yt[j] * p.ld_y + yc, 16);
            return;
        }
        for (int i = tid; i < cnt * NC; i += AD_THREADS) {
            const int col = o * NC + i % NC;
            if (col < p.n_out)
                elem(sm + so + L.b_stage + i / NC * YP + i % NC * (int)sizeof(TO),
                     (const TO *)p.y + (int64_t)s_tok[i / NC] * p.ld_y + col, true, p.y);
        }
    };

    // ---- first product: this CTA's share of n_in, one MT x KW grid of warps
    const int kc = ((int)p.lda + KC - 1) / KC;
    const int k0 = (int)((int64_t)cr * kc / C), k1 = (int)((int64_t)(cr + 1) * kc / C);
    const int mt = warp % MT, kw = warp / MT;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.0f;
    for (int s = 0; s < L.stages - 1; ++s) {
        if (k0 + s < k1) load_k(k0 + s, s);
        cp_commit();
    }
    int stage = 0;
    for (int k = k0; k < k1; ++k) {
        if (L.stages == 3) cp_wait<1>();
        else cp_wait<0>();
        __syncthreads();
        if (k + L.stages - 1 < k1) load_k(k + L.stages - 1, stage == 0 ? L.stages - 1 : stage - 1);
        cp_commit();
        const uint8_t *xs = sm + stage * (L.x_stage + L.a_stage), *as = xs + L.x_stage;
        stage = stage + 1 == L.stages ? 0 : stage + 1;
#pragma unroll
        for (int kk = kw; kk < KC / 16; kk += KW) {
            if constexpr (X16) {
                uint32_t af[4];
                ldm4(af, smem_u32(xs + (16 * mt + (lane & 15)) * XP + 32 * kk + 16 * (lane >> 4)));
#pragma unroll
                for (int n = 0; n < NT; n += 2) {
                    if (n >= nt) break;
                    // rows of two n tiles (the last row again where the second lies past r8)
                    const int r = min(8 * n + (lane & 7) + 8 * (lane >> 4), r8 - 1);
                    uint32_t bf[4];
                    ldm4(bf, smem_u32(as + r * AP + 32 * kk + 16 * (lane >> 3 & 1)));
                    mma16(acc[n], af, bf[0], bf[1], TW());
                    if (n + 1 < nt) mma16(acc[n + 1], af, bf[2], bf[3], TW());
                }
            } else {
                // two k8 steps; the mma's k slots q, q + 4 hold columns 2q, 2q + 1 of both operands
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int col = 16 * kk + 8 * h + 2 * (lane & 3);
                    const float2 u = *reinterpret_cast<const float2 *>(xs + (16 * mt + (lane >> 2)) * XP + 4 * col);
                    const float2 v = *reinterpret_cast<const float2 *>(xs + (16 * mt + 8 + (lane >> 2)) * XP + 4 * col);
                    uint32_t hi[4], lo[4];
                    split(u.x, hi[0], lo[0]);
                    split(v.x, hi[1], lo[1]);
                    split(u.y, hi[2], lo[2]);
                    split(v.y, hi[3], lo[3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (n >= nt) break;
                        uint32_t b0, b1;
                        pair32(*reinterpret_cast<const uint32_t *>(as + (8 * n + (lane >> 2)) * AP + 2 * col), b0, b1, TW());
                        mma8(acc[n], lo, b0, b1);
                        mma8(acc[n], hi, b0, b1);
                    }
                }
            }
        }
    }
    cp_wait<0>();
    __syncthreads();   // the ring is free

    // the first chunks of B travel while the partial sums meet
    for (int s = 0; s < L.b_stages - 1; ++s) {
        if (s0 + s < s1) load_b(s0 + s, s);
        cp_commit();
    }
    // ---- add the KW partial sums of the CTA, then those of the cluster, in order
    {
        const int pitch = p.rank + 8;
        float *red = reinterpret_cast<float *>(sm);   // [KW][M][pitch]
        float *mine = red + (kw * M + 16 * mt + (lane >> 2)) * pitch + 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            if (n >= nt) break;
            *reinterpret_cast<float2 *>(mine + 8 * n) = make_float2(acc[n][0], acc[n][1]);
            *reinterpret_cast<float2 *>(mine + 8 * pitch + 8 * n) = make_float2(acc[n][2], acc[n][3]);
        }
        __syncthreads();
        float *part = reinterpret_cast<float *>(sm + L.off_part);
        {
            constexpr int TR = AD_THREADS / M;         // threads per row, four columns each in turn
            const int m = tid / TR;
            for (int r = 4 * (tid % TR); r < r8; r += 4 * TR) {
                const int at = m * pitch + r;
                float4 v = *reinterpret_cast<const float4 *>(red + at);
#pragma unroll
                for (int w = 1; w < KW; ++w) {
                    const float4 u = *reinterpret_cast<const float4 *>(red + w * M * pitch + at);
                    v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
                }
                *reinterpret_cast<float4 *>(part + at) = v;
            }
        }
        cl.sync();
        // CTA cr adds up its M / C rows and gives the parts to the whole cluster
        const float scale = p.scale[a];
        const int rows = M / C, tr = min(32, AD_THREADS / rows);   // threads per row: a power of two
        const int q = tid & (tr - 1), mr = tid / tr, m = cr * rows + mr;
        if (mr < rows) {   // (whole warps: 32 * C / M rows of them)
            constexpr int RT = 8 * NT / 4 * M / AD_THREADS > 0 ? 8 * NT / 4 * M / AD_THREADS : 1;   // groups of four per thread
            float low[RT][4];
            float top = 0.0f;                                   // the largest finite |low| of the row
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const int r = 4 * (q + j * tr);
#pragma unroll
                for (int e = 0; e < 4; ++e) low[j][e] = 0.0f;
                if (r >= r8) continue;
                float4 u[8];
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c < C) u[c] = *reinterpret_cast<const float4 *>(cl.map_shared_rank(part, c) + m * pitch + r);
#pragma unroll
                for (int c = 0; c < 8; ++c)
                    if (c < C) { low[j][0] += u[c].x; low[j][1] += u[c].y; low[j][2] += u[c].z; low[j][3] += u[c].w; }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    low[j][e] = r + e < rank ? low[j][e] * scale : 0.0f;
                    if (SCALED && fabsf(low[j][e]) < INFINITY) top = fmaxf(top, fabsf(low[j][e]));
                }
            }
            float up = 1.0f;
            if (SCALED) {
                for (int off = tr / 2; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor_sync(MOE_FULL, top, off));
                // 2^e brings the largest into [2^14, 2^15); e within the exponents whose inverse is normal too
                const int e = top > 0.0f ? min(max(14 - ilogbf(top), -126), 126) : 0;
                up = __int_as_float((127 + e) << 23);
                if (q == 0)
                    for (int c = 0; c < C; ++c) cl.map_shared_rank(s_fac, c)[m] = __int_as_float((127 - e) << 23);
            }
#pragma unroll
            for (int j = 0; j < RT; ++j) {
                const int r = 4 * (q + j * tr);
                if (r >= r16) continue;
                uint2 w[P];
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = low[j][e] * up;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    float c[4];   // v, but no finite value rounds to an infinite bf16
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        c[e] = !SCALED && i == 0 && fabsf(v[e]) < INFINITY ? fminf(fmaxf(v[e], -0x1.fep127f), 0x1.fep127f) : v[e];
                    w[i] = ad_pack(c, TW());
                    float h[4];
                    uint32_t b0, b1;
                    pair32(w[i].x, b0, b1, TW());
                    h[0] = __uint_as_float(b0); h[1] = __uint_as_float(b1);
                    pair32(w[i].y, b0, b1, TW());
                    h[2] = __uint_as_float(b0); h[3] = __uint_as_float(b1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = v[e] == h[e] ? 0.0f : v[e] - h[e];   // (inf - inf is no remainder)
                }
                for (int c = 0; c < C; ++c) {
                    uint8_t *dst = cl.map_shared_rank(sm, c) + m * bp + 2 * r;
#pragma unroll
                    for (int i = 0; i < P; ++i) *reinterpret_cast<uint2 *>(dst + i * M * bp) = w[i];
                }
            }
        }
        cl.sync();   // every CTA has all parts
    }

    // ---- second product: [M][rank] x [rank][NC] per step; warps MT x KW over the n tiles.  The
    // products are added to y's tile in shared memory, which is then written out in whole rows.
    constexpr int WN = NC / 8 / KW;   // n tiles per warp
    const int m_lo = 16 * mt + (lane >> 2);
    const float f_lo = SCALED ? s_fac[m_lo] : 1.0f, f_hi = SCALED ? s_fac[m_lo + 8] : 1.0f;
    const uint32_t a_off = sm0 + (16 * mt + (lane & 15)) * bp + 16 * (lane >> 4);
    const uint32_t b_off = (8 * WN * kw + (lane & 7) + 8 * (lane >> 4)) * bp + 16 * (lane >> 3 & 1);
    // the parts of A x are the same in every step: kept in registers up to rank 64
    constexpr bool KEEP = NT <= 8;
    constexpr int KS = KEEP ? NT / 2 : 1;
    uint32_t keep[KS][P][4];
    if (KEEP) {
#pragma unroll
        for (int kk = 0; kk < KS; ++kk)
            if (kk < r16 / 16) {
#pragma unroll
                for (int i = 0; i < P; ++i) ldm4(keep[kk][i], a_off + i * M * bp + 32 * kk);
            }
    }
    stage = 0;
    for (int o = s0; o < s1; ++o) {
        if (L.b_stages == 3) cp_wait<1>();
        else cp_wait<0>();
        __syncthreads();   // chunk o is there, and the chunk before is used up
        if (o + L.b_stages - 1 < s1) load_b(o + L.b_stages - 1, stage == 0 ? L.b_stages - 1 : stage - 1);
        cp_commit();
        const int so = L.off_b + stage * (L.b_stage + L.y_stage);
        stage = stage + 1 == L.b_stages ? 0 : stage + 1;
        float d[WN][4];
#pragma unroll
        for (int n = 0; n < WN; ++n) d[n][0] = d[n][1] = d[n][2] = d[n][3] = 0.0f;
        auto step = [&](int kk, const uint32_t (&af)[P][4]) {
            uint32_t bf[WN / 2][4];
#pragma unroll
            for (int n = 0; n < WN; n += 2) ldm4(bf[n / 2], sm0 + so + b_off + 8 * n * bp + 32 * kk);
#pragma unroll
            for (int i = P - 1; i >= 0; --i)   // the smallest parts first
#pragma unroll
                for (int n = 0; n < WN; ++n) mma16(d[n], af[i], bf[n / 2][2 * (n & 1)], bf[n / 2][2 * (n & 1) + 1], TW());
        };
        if constexpr (KEEP) {
#pragma unroll
            for (int kk = 0; kk < KS; ++kk)
                if (kk < r16 / 16) step(kk, keep[kk]);
        } else {
#pragma unroll 2
            for (int kk = 0; kk < r16 / 16; ++kk) {
                uint32_t af[P][4];
#pragma unroll
                for (int i = 0; i < P; ++i) ldm4(af[i], a_off + i * M * bp + 32 * kk);
                step(kk, af);
            }
        }
        TO *ys = reinterpret_cast<TO *>(sm + so + L.b_stage + m_lo * YP) + 8 * WN * kw + 2 * (lane & 3);
#pragma unroll
        for (int n = 0; n < WN; ++n) {
            ad_add2(ys + 8 * n, d[n][0], d[n][1], f_lo, !p.y);
            ad_add2(ys + 8 * n + 8 * YP / (int)sizeof(TO), d[n][2], d[n][3], f_hi, !p.y);
        }
        __syncthreads();
        if (vec_o && (o + 1) * NC <= p.n_out) {
            const uint8_t *yo = sm + so + L.b_stage + tid / YC * YP + 16 * (tid % YC);
#pragma unroll
            for (int j = 0; j < YN; ++j)
                if (yt[j] >= 0)
                    *reinterpret_cast<uint4 *>((TO *)p.out + (int64_t)yt[j] * p.ld_out + o * NC + YE * (tid % YC)) =
                        *reinterpret_cast<const uint4 *>(yo + j * YR * YP);
            continue;
        }
        for (int i = tid; i < cnt * NC; i += AD_THREADS) {
            const int col = o * NC + i % NC;
            if (col < p.n_out)
                ((TO *)p.out)[(int64_t)s_tok[i / NC] * p.ld_out + col] =
                    *reinterpret_cast<const TO *>(sm + so + L.b_stage + i / NC * YP + i % NC * (int)sizeof(TO));
        }
    }
    cp_wait<0>();
}

template <typename TX, typename TW, typename TO, int M, int NT>
static cudaError_t adapters_launch(const AdapterArgs &p, cudaStream_t s) {
    constexpr int KC = ad_kc<M>(), NC = ad_nc<M>();
    constexpr int P = std::is_same<TW, __nv_bfloat16>::value && sizeof(TO) == 4 ? 3 : 2;
    const int kc = (int)((p.lda + KC - 1) / KC), oc = (p.n_out + NC - 1) / NC;
    // at most one partial tile per adapter in use (and for the rows without one)
    const int64_t tiles = std::min<int64_t>(p.n_tok, ((int64_t)p.n_tok + M - 1) / M + std::min(p.n_adapters + 1, p.n_tok));
    // CTAs per tile: as many as one wave of two per SM holds (320: a few end early), at most one per
    // step of a product.  The grid's bound counts a partial tile for every adapter; about three
    // quarters of that is met.  512 / 2048 tokens, 8 adapters of rank 64, fp32: 8 CTAs 16.6 / 31.0
    // us, 4 CTAs 18.6 / 35.1; 768 tokens: 8 CTAs 28.9 us, 4 CTAs 22.8.
    const int64_t met = std::min<int64_t>(p.n_tok, p.n_tok / M + 1 + 3 * (int64_t)std::min(p.n_adapters + 1, p.n_tok) / 4);
    int C = 1;
    while (C < 8 && met * 2 * C <= 320 && 2 * C <= std::max(kc, oc)) C *= 2;
    AdSmem L{};
    L.x_stage = M * (KC * (int)sizeof(TX) + (sizeof(TX) == 2 ? 16 : 32));
    L.a_stage = p.rank * (KC * 2 + 16);
    const int pitch = p.rank + 8, KW = AD_WARPS / (M / 16), bp = ((p.rank + 15) & ~15) * 2 + 16;
    const int red = KW * M * pitch * 4, low = P * M * bp, part = M * pitch * 4;
    L.off_part = std::max(red, low);
    L.b_stage = NC * bp;
    L.y_stage = M * (NC * (int)sizeof(TO) + (sizeof(TO) == 4 ? 32 : 16));
    // up to three stages each: as many as leave room for a second CTA on the SM, else two, else what fits
    const int ks = std::max(2, std::min(3, kc / C + 1)), bs = std::max(2, std::min(3, oc / C + 1));
    auto lay = [&](int k, int o, int limit) {
        L.stages = k;
        L.b_stages = o;
        L.off_b = std::max(k * (L.x_stage + L.a_stage), L.off_part + part);
        L.off_hist = L.off_b + o * (L.b_stage + L.y_stage);
        L.bytes = L.off_hist + 4 * (p.n_adapters + 1);
        return L.bytes <= limit;
    };
    constexpr int TWO = 111 * 1024, ONE = 226 * 1024;
    if (!lay(ks, bs, TWO) && !lay(2, bs, TWO) && !lay(2, 2, TWO) && !lay(ks, bs, ONE) && !lay(2, 2, ONE))
        return cudaErrorInvalidValue;
    auto al = [](const void *q, int64_t ld, int size) {
        return !q || (((uintptr_t)q | (uintptr_t)(ld * size)) & 15) == 0;
    };
    const int vec_x = al(p.x, p.ld_x, (int)sizeof(TX));
    const int vec_o = al(p.y, p.ld_y, (int)sizeof(TO)) && al(p.out, p.ld_out, (int)sizeof(TO));
    auto *kern = k_adapters<TX, TW, TO, M, NT>;
    static SmemAttr attr;
    const cudaError_t e = attr.need((const void *)kern, L.bytes);
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, (unsigned)(tiles * C), AD_THREADS, L.bytes, s, C, p, L, vec_x, vec_o);
}

template <typename TX, typename TW, typename TO>
static cudaError_t adapters_go(const AdapterArgs &p, cudaStream_t s) {
    // Tiles of 16 rows until there are enough rows to fill larger ones.  2048 -> 2048 columns, 8
    // adapters in runs, rank 16 / 64 in bf16: 1024 tokens take 13.9 / 18.7 us with 16 rows and 14.6 /
    // 20.6 us with 64, 2048 tokens 18.7 / 26.9 and 18.7 / 23.5 us, 4096 tokens 26.5 / 43.3 and 22.8 /
    // 29.9 us.
    if (p.n_tok <= 1536)
        return p.rank <= 32   ? adapters_launch<TX, TW, TO, 16, 4>(p, s)
               : p.rank <= 64 ? adapters_launch<TX, TW, TO, 16, 8>(p, s)
                              : adapters_launch<TX, TW, TO, 16, 16>(p, s);
    return p.rank <= 64 ? adapters_launch<TX, TW, TO, 64, 8>(p, s) : adapters_launch<TX, TW, TO, 64, 16>(p, s);
}

static cudaError_t adapters_chunk(const AdapterArgs &p, int dt_x, int dt_w, int dt_out, cudaStream_t s) {
    if (dt_x == DT_F32 && dt_out == DT_F32)
        return dt_w == DT_BF16 ? adapters_go<float, __nv_bfloat16, float>(p, s) : adapters_go<float, __half, float>(p, s);
    if (dt_x != dt_w || (dt_out != dt_w && dt_out != DT_F32)) return cudaErrorInvalidValue;
    if (dt_w == DT_BF16)
        return dt_out == DT_F32 ? adapters_go<__nv_bfloat16, __nv_bfloat16, float>(p, s)
                                : adapters_go<__nv_bfloat16, __nv_bfloat16, __nv_bfloat16>(p, s);
    return dt_out == DT_F32 ? adapters_go<__half, __half, float>(p, s) : adapters_go<__half, __half, __half>(p, s);
}

cudaError_t launch_adapters(const AdapterArgs &p, int dt_x, int dt_w, int dt_out, cudaStream_t s) {
    // Every CTA reads all ids of its launch to find its tile, so a launch takes up to 8192 tokens: about
    // one wave of two CTAs per SM, and the ids stay a small part of what a CTA reads.
    constexpr int CHUNK = 8192;
    const int64_t sx = dt_x == DT_F32 ? 4 : 2, so = dt_out == DT_F32 ? 4 : 2;
    for (int64_t t = 0; t < p.n_tok; t += CHUNK) {
        AdapterArgs c = p;
        c.n_tok = (int)std::min<int64_t>(CHUNK, p.n_tok - t);
        c.ids = p.ids + t;
        c.x = (const uint8_t *)p.x + t * p.ld_x * sx;
        c.y = p.y ? (const uint8_t *)p.y + t * p.ld_y * so : nullptr;
        c.out = (uint8_t *)p.out + t * p.ld_out * so;
        const cudaError_t e = adapters_chunk(c, dt_x, dt_w, dt_out, s);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace moe
