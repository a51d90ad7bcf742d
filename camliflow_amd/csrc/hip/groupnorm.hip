// Group normalisation with an activation on channels-last maps, forward and backward, gfx950.
//
//   per sample b and group g (C / G channels x P pixels, N values):   m = mean(x),  r = 1 / sqrt(mean((x - m)^2) + eps)
//   z = (x - m) r w[c] + beta[c],   y = act(z)
//   dz = gy act'(z),  xhat = (x - m) r,  dw[c] = sum dz xhat,  dbeta[c] = sum dz,
//   dx = r (w dz - mean_g(w dz) - xhat mean_g(w dz xhat))
//
// Memory: x is [B][P][C] with any pixel pitch and batch stride (a channel slice of a wider map is read in place), y and dx are
// dense.  Both directions read the map twice (sums, then values): the sums of all pixels of a group have to be known before the
// first value can be written.  All arithmetic is fp32, for every element type.
//
//   stats   one workgroup per (sample, chunk of pixels), all channels: thread = 16 bytes of channels x every rows-th pixel.  Each
//           thread sums (x - pivot) and its square about ITS first value, so a mean far from zero costs no digits; threads, channels
//           and chunks are joined as (count, mean, M2) triples in a fixed order -- no atomics, the same bits on every run.
//   small   a group of at most 16384 values whose channels fit whole vectors: one workgroup of 1024 threads per (sample, group) holds it in
//           registers, so one launch and one reading do (1 x 128 x 17 x 30 fp32: 12 -> 6 us on the GPU).
//   apply   the workgroup joins its sample's chunk triples (a few KB from L2) and writes its chunk.  It takes the chunks in the
//           reverse of the order in which stats read them, so that what stats read last is still in the last-level cache.
//   sums    (backward) per channel sum dz and sum dz xhat of a chunk;  finish: joins the chunks per channel and group;
//   dx      as apply; one extra workgroup adds dw / dbeta over the samples.
//
// Bound by memory.  Measured at 16 x 64 x 272 x 480 bf16, SiLU (267 MB; a large copy: 5.1 TB/s, a sum that only reads: 4.0): stats 58 us,
// apply 106 (5.0 TB/s), sums 132 (4.0), finish 5, dx 174 (4.6); at 8 x 128 x 68 x 120 fp32 (36 MB): 10.5, 17, 14.5, 4.6 and 18 us.
#include "typed.h"

namespace {

constexpr int BLOCK = 256;
constexpr int MAX_C = 4096;

struct GnArgs {
    const void* x;
    int64_t x_bs, x_ld;       // batch stride and pixel pitch, elements
    const void *weight, *bias;
    int wtype;
    int C, G, P, chunks, chunk_px, act;
    bool stream;              // the map is larger than the caches: its second reading and the result are not kept in them
    float eps;
};

// e = exp(-|z|): with it sigmoid(|z|) = 1 / (1 + e) and its complement e / (1 + e) lose no digits where the sigmoid saturates.  fp32 maps
// carry the rounding of the product along (plain exp2(-|z| log2 e) is off by |z| 2^-24).
template <typename T>
__device__ __forceinline__ float exp_minus(float z) {
    constexpr float L = 1.44269502162933349609375f, L_REST = 1.92596299e-8f;      // log2 e
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_exp2f(-fabsf(z) * L);
    } else {
        const float a = fabsf(z), x = a > 87.0f ? -87.0f : -a;
        const float t = x * L, rest = __builtin_fmaf(x, L_REST, __builtin_fmaf(x, L, -t));
        const float e = __builtin_amdgcn_exp2f(t);
        return __builtin_fmaf(e, rest * 0.693147181f, e);
    }
}

template <typename T>
__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case 1: return z > 0.0f || z != z ? z : 0.0f;
        case 2: return z > 0.0f ? z : 0.1f * z;
        case 3: { const float e = exp_minus<T>(z); return (z < 0.0f ? e : 1.0f) * __builtin_amdgcn_rcpf(1.0f + e); }
        case 6: { const float e = exp_minus<T>(z); return z * ((z < 0.0f ? e : 1.0f) * __builtin_amdgcn_rcpf(1.0f + e)); }
        default: return z;
    }
}

template <typename T>
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case 1: return z > 0.0f ? 1.0f : 0.0f;
        case 2: return z > 0.0f ? 1.0f : 0.1f;
        case 3: { const float e = exp_minus<T>(z), r = __builtin_amdgcn_rcpf(1.0f + e); return e * r * r; }
        case 6: {
            const float e = exp_minus<T>(z), r = __builtin_amdgcn_rcpf(1.0f + e), er = e * r;
            return (z < 0.0f ? er : r) * __builtin_fmaf(z, z < 0.0f ? r : er, 1.0f);
        }
        default: return 1.0f;
    }
}

// mean and M2 of the union of NA values (mean, m2) and nb values (mb, qb)
__device__ __forceinline__ void join_moments(float& n, float& mean, float& m2, float nb, float mb, float qb) {
    const float t = n + nb;
    if (nb == 0.0f) return;
    const float d = mb - mean, f = nb / t;
    mean = __builtin_fmaf(d, f, mean);
    m2 += __builtin_fmaf(d * d, n * f, qb);
    n = t;
}

// dynamic LDS: chan float2[C], red float2[BLOCK * VEC]
template <typename T, int VEC>
__global__ __launch_bounds__(BLOCK) void gn_stats_kernel(GnArgs a, float2* __restrict__ partial) {
    extern __shared__ float2 smem[];
    float2* chan = smem;
    float2* red = smem + a.C;
    const int b = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    const int p0 = chunk * a.chunk_px, len = min(a.P - p0, a.chunk_px);
    const T* xb = static_cast<const T*>(a.x) + b * a.x_bs + (int64_t)p0 * a.x_ld;
    const int cv = a.C / VEC;
    for (int c0 = 0; c0 < cv; c0 += BLOCK) {
        const int w = min(BLOCK, cv - c0), rows = BLOCK / w;
        const int r = tid / w, col = tid - r * w;
        if (r < rows) {
            float pivot[VEC], s[VEC], q[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) { pivot[e] = 0.0f; s[e] = 0.0f; q[e] = 0.0f; }
            const T* px = xb + (c0 + col) * VEC;
            const int n = r < len ? (len - r + rows - 1) / rows : 0;
            if (n > 0) load_f32<T, VEC>(px + (int64_t)r * a.x_ld, pivot);
#pragma unroll 4
            for (int i = 1; i < n; ++i) {
                float v[VEC];
                load_f32<T, VEC>(px + (int64_t)(r + i * rows) * a.x_ld, v);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float d = v[e] - pivot[e];
                    s[e] += d;
                    q[e] = __builtin_fmaf(d, d, q[e]);
                }
            }
            const float inv = n > 0 ? 1.0f / (float)n : 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                red[(r * w + col) * VEC + e] = make_float2(__builtin_fmaf(s[e], inv, pivot[e]), q[e] - s[e] * s[e] * inv);
        }
        __syncthreads();
        for (int c = tid; c < w * VEC; c += BLOCK) {
            float n = 0.0f, mean = 0.0f, m2 = 0.0f;
            for (int rr = 0; rr < rows && rr < len; ++rr) {
                const float2 t = red[rr * w * VEC + c];
                join_moments(n, mean, m2, (float)((len - rr + rows - 1) / rows), t.x, t.y);
            }
            chan[c0 * VEC + c] = make_float2(mean, m2);
        }
        __syncthreads();
    }
    const int cpg = a.C / a.G, wave = tid >> 6, lane = tid & 63;
    for (int g = wave; g < a.G; g += BLOCK / 64) {
        float sum = 0.0f;
        for (int c = lane; c < cpg; c += 64) sum += chan[g * cpg + c].x;
        const float mean = wave_sum(sum) / (float)cpg;
        float m2 = 0.0f;
        for (int c = lane; c < cpg; c += 64) {
            const float2 t = chan[g * cpg + c];
            const float d = t.x - mean;
            m2 += __builtin_fmaf(d * d, (float)len, t.y);
        }
        m2 = wave_sum(m2);
        if (lane == 0) partial[((int64_t)b * a.chunks + chunk) * a.G + g] = make_float2(mean, m2);
    }
}

// joins the chunk moments of sample b into stat[g] = (mean, rstd); called by all threads, ends with a barrier
__device__ __forceinline__ void join_chunks(const GnArgs& a, const float2* __restrict__ partial, int b, float2* stat) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const float2* pb = partial + (int64_t)b * a.chunks * a.G;
    const float cpg = (float)(a.C / a.G), total = (float)a.P;
    for (int g = wave; g < a.G; g += BLOCK / 64) {
        float sum = 0.0f;
        for (int i = lane; i < a.chunks; i += 64) sum = __builtin_fmaf(pb[i * a.G + g].x, (float)min(a.P - i * a.chunk_px, a.chunk_px) / total, sum);
        const float mean = wave_sum(sum);
        float m2 = 0.0f;
        for (int i = lane; i < a.chunks; i += 64) {
            const float2 t = pb[i * a.G + g];
            const float d = t.x - mean;
            m2 += __builtin_fmaf(d * d, (float)min(a.P - i * a.chunk_px, a.chunk_px) * cpg, t.y);
        }
        m2 = wave_sum(m2);
        if (lane == 0) stat[g] = make_float2(mean, 1.0f / sqrtf(m2 / (total * cpg) + a.eps));
    }
    __syncthreads();
}

// dynamic LDS: stat float2[G]
template <typename T, int VEC>
__global__ __launch_bounds__(BLOCK) void gn_apply_kernel(GnArgs a, const float2* __restrict__ partial, T* __restrict__ y,
                                                         float2* __restrict__ stat_out) {
    extern __shared__ float2 smem[];
    const int b = gridDim.y - 1 - blockIdx.y, chunk = gridDim.x - 1 - blockIdx.x, tid = threadIdx.x;
    join_chunks(a, partial, b, smem);
    if (stat_out && chunk == 0)
        for (int g = tid; g < a.G; g += BLOCK) stat_out[(int64_t)b * a.G + g] = smem[g];
    const int p0 = chunk * a.chunk_px, len = min(a.P - p0, a.chunk_px);
    const T* xb = static_cast<const T*>(a.x) + b * a.x_bs + (int64_t)p0 * a.x_ld;
    T* yb = y + ((int64_t)b * a.P + p0) * a.C;
    const int cv = a.C / VEC, cpg = a.C / a.G;
    for (int c0 = 0; c0 < cv; c0 += BLOCK) {
        const int w = min(BLOCK, cv - c0), rows = BLOCK / w;
        const int r = tid / w, col = tid - r * w;
        if (r >= rows) continue;
        float mean[VEC], scale[VEC], shift[VEC];
        const int c = (c0 + col) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float2 st = smem[(c + e) / cpg];
            mean[e] = st.x;
            scale[e] = a.weight ? st.y * load_param(a.weight, a.wtype, c + e) : st.y;
            shift[e] = a.bias ? load_param(a.bias, a.wtype, c + e) : 0.0f;
        }
#pragma unroll 4
        for (int p = r; p < len; p += rows) {
            float v[VEC];
            load_f32<T, VEC>(xb + (int64_t)p * a.x_ld + c, v, a.stream);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = act_value<T>(__builtin_fmaf(v[e] - mean[e], scale[e], shift[e]), a.act);
            store_f32<T, VEC>(yb + (int64_t)p * a.C + c, v, a.stream);
        }
    }
}

constexpr int SMALL_THREADS = 1024, SMALL_VALUES = 16;       // per thread

__device__ __forceinline__ float block_sum_1024(float v, float* red) {
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = red[threadIdx.x & 15];
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) t += __shfl_xor(t, off, CAMLI_WAVE);
    __syncthreads();
    return t;
}

// grid (G, B)
template <typename T, int VEC>
__global__ __launch_bounds__(SMALL_THREADS) void gn_small_kernel(GnArgs a, T* __restrict__ y, float2* __restrict__ stat_out) {
    __shared__ float red[SMALL_THREADS / 64];
    constexpr int N = SMALL_VALUES / VEC;
    const int g = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, cpg = a.C / a.G;
    const int w = cpg / VEC, rows = SMALL_THREADS / w, r = tid / w, c = g * cpg + (tid - r * w) * VEC;
    const T* xb = static_cast<const T*>(a.x) + b * a.x_bs + c;
    float v[N][VEC], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int p = r + i * rows;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = 0.0f;
        if (r < rows && p < a.P) load_f32<T, VEC>(xb + (int64_t)p * a.x_ld, v[i]);
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sum += v[i][e];
    const float n = (float)a.P * (float)cpg, mean = block_sum_1024(sum, red) / n;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (r < rows && r + i * rows < a.P) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[i][e] -= mean;
                sum = __builtin_fmaf(v[i][e], v[i][e], sum);
            }
        }
    const float rstd = 1.0f / sqrtf(block_sum_1024(sum, red) / n + a.eps);
    if (stat_out && tid == 0) stat_out[(int64_t)b * a.G + g] = make_float2(mean, rstd);
    if (r >= rows) return;
    float scale[VEC], shift[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        scale[e] = a.weight ? rstd * load_param(a.weight, a.wtype, c + e) : rstd;
        shift[e] = a.bias ? load_param(a.bias, a.wtype, c + e) : 0.0f;
    }
    T* yb = y + (int64_t)b * a.P * a.C + c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int p = r + i * rows;
        if (p >= a.P) break;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = act_value<T>(__builtin_fmaf(v[i][e], scale[e], shift[e]), a.act);
        store_f32<T, VEC>(yb + (int64_t)p * a.C, v[i]);
    }
}

// backward, first pass: csum[b][chunk][c] = (sum dz, sum dz xhat) of the chunk.  dynamic LDS: red float2[BLOCK * VEC]
template <typename T, int VEC>
__global__ __launch_bounds__(BLOCK) void gn_bwd_sums_kernel(GnArgs a, const T* __restrict__ gy, const float2* __restrict__ stat,
                                                            float2* __restrict__ csum) {
    extern __shared__ float2 red[];
    const int b = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
    const int p0 = chunk * a.chunk_px, len = min(a.P - p0, a.chunk_px);
    const T* xb = static_cast<const T*>(a.x) + b * a.x_bs + (int64_t)p0 * a.x_ld;
    const T* gb = gy + ((int64_t)b * a.P + p0) * a.C;
    float2* out = csum + ((int64_t)b * a.chunks + chunk) * a.C;
    const int cv = a.C / VEC, cpg = a.C / a.G;
    for (int c0 = 0; c0 < cv; c0 += BLOCK) {
        const int w = min(BLOCK, cv - c0), rows = BLOCK / w;
        const int r = tid / w, col = tid - r * w;
        if (r < rows) {
            float mean[VEC], rstd[VEC], wt[VEC], shift[VEC], s0[VEC], s1[VEC];
            const int c = (c0 + col) * VEC;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 st = stat[(int64_t)b * a.G + (c + e) / cpg];
                mean[e] = st.x;
                rstd[e] = st.y;
                wt[e] = a.weight ? load_param(a.weight, a.wtype, c + e) : 1.0f;
                shift[e] = a.bias ? load_param(a.bias, a.wtype, c + e) : 0.0f;
                s0[e] = 0.0f;
                s1[e] = 0.0f;
            }
#pragma unroll 2
            for (int p = r; p < len; p += rows) {
                float v[VEC], g[VEC];
                load_f32<T, VEC>(xb + (int64_t)p * a.x_ld + c, v);
                load_f32<T, VEC>(gb + (int64_t)p * a.C + c, g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float xhat = (v[e] - mean[e]) * rstd[e];
                    const float dz = g[e] * act_slope<T>(__builtin_fmaf(v[e] - mean[e], rstd[e] * wt[e], shift[e]), a.act);
                    s0[e] += dz;
                    s1[e] = __builtin_fmaf(dz, xhat, s1[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) red[(r * w + col) * VEC + e] = make_float2(s0[e], s1[e]);
        }
        __syncthreads();
        for (int c = tid; c < w * VEC; c += BLOCK) {
            float t0 = 0.0f, t1 = 0.0f;
            for (int rr = 0; rr < rows; ++rr) {
                const float2 t = red[rr * w * VEC + c];
                t0 += t.x;
                t1 += t.y;
            }
            out[c0 * VEC + c] = make_float2(t0, t1);
        }
        __syncthreads();
    }
}

// joins the chunks: csum2[b][c], and per group gmean[b][g] = (mean(w dz), mean(w dz xhat)).  grid (G, B)
__global__ __launch_bounds__(BLOCK) void gn_bwd_finish_kernel(GnArgs a, const float2* __restrict__ csum, float2* __restrict__ csum2,
                                                              float2* __restrict__ gmean) {
    __shared__ float2 acc[BLOCK / 64];
    const int g = blockIdx.x, b = blockIdx.y, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, cpg = a.C / a.G;
    float g0 = 0.0f, g1 = 0.0f;
    for (int c = g * cpg + wave; c < (g + 1) * cpg; c += BLOCK / 64) {
        float s0 = 0.0f, s1 = 0.0f;
        for (int i = lane; i < a.chunks; i += 64) {
            const float2 t = csum[((int64_t)b * a.chunks + i) * a.C + c];
            s0 += t.x;
            s1 += t.y;
        }
        s0 = wave_sum(s0);
        s1 = wave_sum(s1);
        if (lane == 0) csum2[(int64_t)b * a.C + c] = make_float2(s0, s1);
        const float wt = a.weight ? load_param(a.weight, a.wtype, c) : 1.0f;
        g0 = __builtin_fmaf(wt, s0, g0);
        g1 = __builtin_fmaf(wt, s1, g1);
    }
    if (lane == 0) acc[wave] = make_float2(g0, g1);
    __syncthreads();
    if (threadIdx.x == 0) {
        const float inv = 1.0f / ((float)a.P * (float)cpg);
        gmean[(int64_t)b * a.G + g] = make_float2(((acc[0].x + acc[1].x) + (acc[2].x + acc[3].x)) * inv,
                                                  ((acc[0].y + acc[1].y) + (acc[2].y + acc[3].y)) * inv);
    }
}

// grid (chunks + 1, B): the last column of workgroups (sample 0's) sums dw / dbeta over the samples
template <typename T, int VEC>
__global__ __launch_bounds__(BLOCK) void gn_bwd_dx_kernel(GnArgs a, const T* __restrict__ gy, const float2* __restrict__ stat,
                                                          const float2* __restrict__ csum2, const float2* __restrict__ gmean,
                                                          T* __restrict__ gx, float* __restrict__ gw, float* __restrict__ gb_out, int B) {
    const int tid = threadIdx.x;
    if ((int)blockIdx.x == a.chunks) {
        if (blockIdx.y != 0) return;
        for (int c = tid; c < a.C; c += BLOCK) {
            float s0 = 0.0f, s1 = 0.0f;
            for (int b = 0; b < B; ++b) {
                const float2 t = csum2[(int64_t)b * a.C + c];
                s0 += t.x;
                s1 += t.y;
            }
            if (gw) gw[c] = s1;
            if (gb_out) gb_out[c] = s0;
        }
        return;
    }
    if (!gx) return;
    const int b = gridDim.y - 1 - blockIdx.y, chunk = a.chunks - 1 - blockIdx.x;
    const int p0 = chunk * a.chunk_px, len = min(a.P - p0, a.chunk_px);
    const T* xb = static_cast<const T*>(a.x) + b * a.x_bs + (int64_t)p0 * a.x_ld;
    const int64_t dense = ((int64_t)b * a.P + p0) * a.C;
    const int cv = a.C / VEC, cpg = a.C / a.G;
    for (int c0 = 0; c0 < cv; c0 += BLOCK) {
        const int w = min(BLOCK, cv - c0), rows = BLOCK / w;
        const int r = tid / w, col = tid - r * w;
        if (r >= rows) continue;
        float mean[VEC], rstd[VEC], wt[VEC], shift[VEC], m0[VEC], m1[VEC];
        const int c = (c0 + col) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int64_t g = (int64_t)b * a.G + (c + e) / cpg;
            const float2 st = stat[g], gm = gmean[g];
            mean[e] = st.x;
            rstd[e] = st.y;
            wt[e] = a.weight ? load_param(a.weight, a.wtype, c + e) : 1.0f;
            shift[e] = a.bias ? load_param(a.bias, a.wtype, c + e) : 0.0f;
            m0[e] = gm.x;
            m1[e] = gm.y;
        }
#pragma unroll 2
        for (int p = r; p < len; p += rows) {
            float v[VEC], g[VEC];
            load_f32<T, VEC>(xb + (int64_t)p * a.x_ld + c, v, a.stream);
            load_f32<T, VEC>(gy + dense + (int64_t)p * a.C + c, g, a.stream);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float d = v[e] - mean[e], xhat = d * rstd[e];
                const float dz = g[e] * act_slope<T>(__builtin_fmaf(d, rstd[e] * wt[e], shift[e]), a.act);
                v[e] = rstd[e] * (__builtin_fmaf(wt[e], dz, -m0[e]) - xhat * m1[e]);
            }
            store_f32<T, VEC>(gx + dense + (int64_t)p * a.C + c, v, a.stream);
        }
    }
}

// Chunks per sample.  A workgroup has a fixed cost (its tree of sums, in apply the joining of its sample's chunk moments), a small map needs
// workgroups more than long ones: 32 KB of the map each, but 256 workgroups at least and 2048 at most, none below 8 KB, and at most 256
// a sample.  (8 x 128 x 68 x 120 fp32, 36 MB: apply 24 us with 2048 workgroups, 17 with 1024; 267 MB: stats 58 us with 2048, 75 with 1024.)
int gn_chunk_px(int B, int C, int P, int type) {
    const int64_t px_bytes = (int64_t)C * camli_type_size(type), total = px_bytes * P * B;
    int64_t want = total >> 15;
    want = want < 256 ? 256 : want > 2048 ? 2048 : want;
    want = (want + B - 1) / B < 256 ? (want + B - 1) / B : 256;
    int64_t px = (8192 + px_bytes - 1) / px_bytes;
    const int64_t even = (P + want - 1) / want;
    if (px < even) px = even;
    return (int)(px < P ? px : P);
}

// in 64 bits: a chunk is a 256th of the map at least, and P + that passes 2^31 from 2^31 - 2^23 positions on
int gn_chunks(int P, int chunk_px) { return (int)(((int64_t)P + chunk_px - 1) / chunk_px); }

bool gn_args_ok(int B, int C, int G, int P, int type, int wtype, int act, const char* who) {
    if (B < 1 || B > 65535 || P < 1 || C < 1 || C > MAX_C || G < 1 || C % G != 0 || type < 0 || type > 2 || wtype < 0 || wtype > 2 ||
        !(act == 0 || act == 1 || act == 2 || act == 3 || act == 6)) {
        camli_set_error("%s: need 1 <= B <= 65535, P >= 1, 1 <= C <= %d, G dividing C, types 0..2, act 0/1/2/3/6 (B=%d C=%d G=%d P=%d type=%d wtype=%d act=%d)",
                        who, MAX_C, B, C, G, P, type, wtype, act);
        return false;
    }
    return true;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

GnArgs make_args(const void* x, int64_t x_bs, int64_t x_ld, const void* weight, const void* bias, int wtype, int B, int C, int G, int P,
                 float eps, int act, int type) {
    GnArgs a;
    a.x = x; a.x_bs = x_bs; a.x_ld = x_ld; a.weight = weight; a.bias = bias; a.wtype = wtype;
    a.C = C; a.G = G; a.P = P; a.act = act; a.eps = eps;
    a.chunk_px = gn_chunk_px(B, C, P, type);
    a.chunks = gn_chunks(P, a.chunk_px);
    // half of the 256 MB last-level cache.  At 16 x 64 x 272 x 480 bf16 (267 MB) keeping nothing of the result leaves what the first
    // reading brought for the second: 196 -> 161 us forward, 305 -> 285 us backward; a smaller map is left for its next reader.
    a.stream = (int64_t)B * P * C * camli_type_size(type) >= ((int64_t)128 << 20);
    return a;
}

template <typename T, int VEC>
int run_fwd(const GnArgs& a, void* y, float2* stat, float2* partial, int B, hipStream_t s) {
    const int cpg = a.C / a.G, w = cpg / VEC;
    if (cpg % VEC == 0 && w <= SMALL_THREADS && (int64_t)a.P <= (int64_t)(SMALL_THREADS / w) * (SMALL_VALUES / VEC)) {
        gn_small_kernel<T, VEC><<<dim3(a.G, B), SMALL_THREADS, 0, s>>>(a, static_cast<T*>(y), stat);
        return camli_check_launch("camli_group_norm_fwd");
    }
    const size_t lds = sizeof(float2) * ((size_t)a.C + BLOCK * VEC);
    gn_stats_kernel<T, VEC><<<dim3(a.chunks, B), BLOCK, lds, s>>>(a, partial);
    gn_apply_kernel<T, VEC><<<dim3(a.chunks, B), BLOCK, sizeof(float2) * a.G, s>>>(a, partial, static_cast<T*>(y), stat);
    return camli_check_launch("camli_group_norm_fwd");
}

template <typename T, int VEC>
int run_bwd(const GnArgs& a, const void* gy, const float2* stat, float2* ws, void* gx, float* gw, float* gb, int B, hipStream_t s) {
    float2 *csum = ws, *csum2 = csum + (size_t)B * a.chunks * a.C, *gmean = csum2 + (size_t)B * a.C;
    gn_bwd_sums_kernel<T, VEC><<<dim3(a.chunks, B), BLOCK, sizeof(float2) * BLOCK * VEC, s>>>(a, static_cast<const T*>(gy), stat, csum);
    gn_bwd_finish_kernel<<<dim3(a.G, B), BLOCK, 0, s>>>(a, csum, csum2, gmean);
    gn_bwd_dx_kernel<T, VEC><<<dim3(a.chunks + 1, B), BLOCK, 0, s>>>(a, static_cast<const T*>(gy), stat, csum2, gmean, static_cast<T*>(gx), gw, gb, B);
    return camli_check_launch("camli_group_norm_bwd");
}

// 16-byte accesses need whole vectors of channels and 16-byte aligned rows; anything else goes element by element
bool vector_ok(const GnArgs& a, int type, const void* p0, const void* p1) {
    const int vec = 16 / camli_type_size(type);
    return a.C % vec == 0 && a.x_ld % vec == 0 && a.x_bs % vec == 0 && aligned16(a.x) && aligned16(p0) && aligned16(p1);
}

}  // namespace

extern "C" int64_t camli_group_norm_fwd_workspace_bytes(int B, int C, int G, int P, int type) {
    if (!gn_args_ok(B, C, G, P, type, 0, 0, "camli_group_norm_fwd_workspace_bytes")) return 0;
    return (int64_t)sizeof(float2) * B * gn_chunks(P, gn_chunk_px(B, C, P, type)) * G;
}

extern "C" int64_t camli_group_norm_bwd_workspace_bytes(int B, int C, int G, int P, int type) {
    if (!gn_args_ok(B, C, G, P, type, 0, 0, "camli_group_norm_bwd_workspace_bytes")) return 0;
    return (int64_t)sizeof(float2) * B * ((int64_t)gn_chunks(P, gn_chunk_px(B, C, P, type)) * C + C + G);
}

extern "C" int camli_group_norm_fwd(const void* x, int64_t x_batch_stride, int64_t x_pixel_stride, const void* weight, const void* bias,
                                    int wtype, void* y, float* stat, void* workspace, int64_t workspace_bytes, int B, int C, int G, int P,
                                    float eps, int act, int type, void* stream) {
    if (!gn_args_ok(B, C, G, P, type, wtype, act, "camli_group_norm_fwd")) return CAMLI_EINVAL;
    if (!x || !y || !workspace || workspace_bytes < camli_group_norm_fwd_workspace_bytes(B, C, G, P, type)) {
        camli_set_error("camli_group_norm_fwd: null pointer or workspace too small");
        return CAMLI_EINVAL;
    }
    const GnArgs a = make_args(x, x_batch_stride, x_pixel_stride, weight, bias, wtype, B, C, G, P, eps, act, type);
    const bool vec = vector_ok(a, type, y, y);
    hipStream_t s = static_cast<hipStream_t>(stream);
    float2 *st = reinterpret_cast<float2*>(stat), *ws = static_cast<float2*>(workspace);
    if (type == CAMLI_F32) return vec ? run_fwd<float, 4>(a, y, st, ws, B, s) : run_fwd<float, 1>(a, y, st, ws, B, s);
    if (type == CAMLI_BF16) return vec ? run_fwd<__bf16, 8>(a, y, st, ws, B, s) : run_fwd<__bf16, 1>(a, y, st, ws, B, s);
    return vec ? run_fwd<_Float16, 8>(a, y, st, ws, B, s) : run_fwd<_Float16, 1>(a, y, st, ws, B, s);
}

extern "C" int camli_group_norm_bwd(const void* gy, const void* x, int64_t x_batch_stride, int64_t x_pixel_stride, const void* weight,
                                    const void* bias, int wtype, const float* stat, void* gx, float* gw, float* gb, void* workspace,
                                    int64_t workspace_bytes, int B, int C, int G, int P, int act, int type, void* stream) {
    if (!gn_args_ok(B, C, G, P, type, wtype, act, "camli_group_norm_bwd")) return CAMLI_EINVAL;
    if (!gy || !x || !stat || !workspace || workspace_bytes < camli_group_norm_bwd_workspace_bytes(B, C, G, P, type)) {
        camli_set_error("camli_group_norm_bwd: null pointer or workspace too small");
        return CAMLI_EINVAL;
    }
    const GnArgs a = make_args(x, x_batch_stride, x_pixel_stride, weight, bias, wtype, B, C, G, P, 0.0f, act, type);
    const bool vec = vector_ok(a, type, gy, gx ? gx : gy);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const float2* st = reinterpret_cast<const float2*>(stat);
    float2* ws = static_cast<float2*>(workspace);
    if (type == CAMLI_F32) return vec ? run_bwd<float, 4>(a, gy, st, ws, gx, gw, gb, B, s) : run_bwd<float, 1>(a, gy, st, ws, gx, gw, gb, B, s);
    if (type == CAMLI_BF16) return vec ? run_bwd<__bf16, 8>(a, gy, st, ws, gx, gw, gb, B, s) : run_bwd<__bf16, 1>(a, gy, st, ws, gx, gw, gb, B, s);
    return vec ? run_bwd<_Float16, 8>(a, gy, st, ws, gx, gw, gb, B, s) : run_bwd<_Float16, 1>(a, gy, st, ws, gx, gw, gb, B, s);
}
