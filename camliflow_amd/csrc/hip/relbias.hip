// The bucketed relative position bias as a tensor, with the gradient of its table, gfx950 (definition: relbias.h).
//
// Forward: bound by writing [B, H, Lq, Lk]; a thread keeps the key positions of its 16 bytes of columns in registers over 32 rows.
// Backward: bound by reading the incoming gradient once.  dtable[a, n, h] adds up to millions of elements into each of a few dozen
// places; every thread adds to a column of an LDS histogram that no other one adds to at the same time (one axis: its own; two: hist_add2), so
// the order of every sum is fixed by the sizes alone and plain reads and writes do.  Columns are added in a fixed order at the end, workgroups in 64 bits.
// Measured at 4 heads x 2048 x 8160, two axes of 32 buckets, bf16 (134 MB): forward 30 us (4.5 TB/s), gradient 64 us (two dependent LDS
// read-add-writes an element) and 4 us for the join; 4 x 501 x 1237, one axis, fp32: 10, 12 and 4 us.
#include "relbias.h"

#include <math.h>

namespace {

constexpr int BLOCK = 256;
constexpr int ROWS = 32;        // rows of the bias a workgroup writes per column tile

constexpr int bwd_columns(int axes) { return axes > 1 ? BLOCK / 2 : BLOCK; }        // of the gradient's histogram

// dynamic LDS: float[axes][2 limit + 1].  grid (column tiles, row tiles, B * H)
template <typename T, int VEC, int AXES>
__global__ __launch_bounds__(BLOCK) void rel_bias_fwd_kernel(RelBias r, T* __restrict__ out, int H, int Lq, int Lk, int cols) {
    extern __shared__ float tab[];
    const int h = blockIdx.z % H, b = blockIdx.z / H, tid = threadIdx.x, span = 2 * r.limit + 1;
    const int* border = rel_stage_borders(r);
    for (int i = tid; i < span; i += BLOCK) {
        const int n = rel_bucket(r, border, i);
#pragma unroll
        for (int a = 0; a < AXES; ++a) tab[a * span + i] = load_param(r.table, r.type, (int64_t)(a * r.buckets + n) * H + h);
    }
    __syncthreads();
    const int tx = tid % cols, ty = tid / cols, per = BLOCK / cols;
    const int j = (blockIdx.x * cols + tx) * VEC;
    if (j >= Lk) return;
    int kp[AXES][VEC], lo[AXES], hi[AXES];
    const int* kpos = r.kpos + b * r.kpos_bs;
    const int* qpos = r.qpos + b * r.qpos_bs;
#pragma unroll
    for (int a = 0; a < AXES; ++a) {
        const int centre = (int)lds_address(tab + a * span + r.limit);
        lo[a] = centre - 4 * r.limit;
        hi[a] = centre + 4 * r.limit;
#pragma unroll
        for (int e = 0; e < VEC; ++e) kp[a][e] = centre + scale_pos<4>(kpos[(int64_t)(j + e) * AXES + a]);
    }
    const int i1 = min(Lq, ((int)blockIdx.y + 1) * ROWS * per);
    for (int i = blockIdx.y * ROWS * per + ty; i < i1; i += per) {
        float v[VEC];
        int qp[AXES];
#pragma unroll
        for (int a = 0; a < AXES; ++a) qp[a] = scale_pos<4>(qpos[(int64_t)i * AXES + a]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[e] = lds_load<float>(med3(kp[0][e] - qp[0], lo[0], hi[0]));
            if (AXES > 1) v[e] += lds_load<float>(med3(kp[AXES - 1][e] - qp[AXES - 1], lo[AXES - 1], hi[AXES - 1]));
        }
        store_f32<T, VEC>(out + ((int64_t)blockIdx.z * Lq + i) * Lk + j, v);
    }
}

// dynamic LDS: float hist[axes * buckets][columns], then unsigned short bucket[2 limit + 1] (two bytes an entry: the usual tables fit one
// dword per bank, so lanes with different offsets do not collide).
// One axis: a column per thread.  Two: lanes l and l + 32 of a wave share one.  They take the axes in opposite order, so at any time one of
// them is among the rows of the first axis and the other among those of the second: half the LDS, twice the workgroups on a CU to cover
// the way of a cell from LDS and back (4 heads x 2048 x 8160 bf16: 73 -> 64 us).
// grid (row parts, column tiles, H): as in the forward a thread keeps its columns' positions in registers and walks over rows; the next
// row's gradient is on its way while one is added.
template <typename T, int VEC, int AXES>
__global__ __launch_bounds__(BLOCK) void rel_bias_bwd_kernel(RelBias r, const T* __restrict__ g, float* __restrict__ partial, int H, int Lq,
                                                             int Lk, int64_t rows, int cols) {
    extern __shared__ float hist[];
    constexpr int COLS = bwd_columns(AXES);
    const int h = blockIdx.z, tid = threadIdx.x, span = 2 * r.limit + 1, nrows = AXES * r.buckets;
    const int half = AXES > 1 ? (tid >> 5) & 1 : 0;             // a thread's axis in turn x is x ^ half
    unsigned short* bucket = reinterpret_cast<unsigned short*>(hist + nrows * COLS);
    const int* border = rel_stage_borders(r);
    for (int i = tid; i < span; i += BLOCK) bucket[i] = (unsigned short)rel_bucket(r, border, i);
    for (int i = tid; i < nrows * COLS; i += BLOCK) hist[i] = 0.0f;
    __syncthreads();
    unsigned column[AXES];
#pragma unroll
    for (int a = 0; a < AXES; ++a) column[a] = ((a ^ half) * r.buckets * COLS + (AXES > 1 ? (tid >> 6) * 32 + (tid & 31) : tid)) * (unsigned)sizeof(float);
    char* cells = reinterpret_cast<char*>(hist);
    const int tx = tid % cols, ty = tid / cols, per = BLOCK / cols, j = (blockIdx.y * cols + tx) * VEC;
    const int64_t first = (int64_t)blockIdx.x * per + ty;
    const int step = gridDim.x * per, step_b = step / Lq, step_i = step - step_b * Lq;
    if (j < Lk && first < rows) {
        const int centre = (int)lds_address(bucket + r.limit), lo = centre - 2 * r.limit, hi = centre + 2 * r.limit, B = (int)(rows / Lq);
        int b = (int)(first / Lq), i = (int)(first - (int64_t)b * Lq), of = -1;      // of: the sample whose positions kp holds
        int kp[AXES][VEC], q[AXES];
        float v[VEC];
        load_f32<T, VEC>(g + (((int64_t)b * H + h) * Lq + i) * Lk + j, v);
#pragma unroll
        for (int a = 0; a < AXES; ++a) q[a] = r.qpos[b * r.qpos_bs + (int64_t)i * AXES + (a ^ half)];
        while (b < B) {
            float now[VEC];
            int qs[AXES];
            const int sample = b;
#pragma unroll
            for (int e = 0; e < VEC; ++e) now[e] = v[e];
#pragma unroll
            for (int a = 0; a < AXES; ++a) qs[a] = scale_pos<2>(q[a]);
            b += step_b;
            i += step_i;
            if (i >= Lq) {
                i -= Lq;
                ++b;
            }
            if (b < B) {
                load_f32<T, VEC>(g + (((int64_t)b * H + h) * Lq + i) * Lk + j, v);
#pragma unroll
                for (int a = 0; a < AXES; ++a) q[a] = r.qpos[b * r.qpos_bs + (int64_t)i * AXES + (a ^ half)];
            }
            if (sample != of) {
                of = sample;
#pragma unroll
                for (int a = 0; a < AXES; ++a)
#pragma unroll
                    for (int e = 0; e < VEC; ++e) kp[a][e] = centre + scale_pos<2>(r.kpos[sample * r.kpos_bs + (int64_t)(j + e) * AXES + (a ^ half)]);
            }
            unsigned n[AXES][VEC];
#pragma unroll
            for (int a = 0; a < AXES; ++a)
#pragma unroll
                for (int e = 0; e < VEC; ++e) n[a][e] = lds_load<unsigned short>(med3(kp[a][e] - qs[a], lo, hi)) * (COLS * (unsigned)sizeof(float)) + column[a];
#pragma unroll
            for (int a = 0; a < AXES; ++a) {
                if constexpr (VEC > 1) {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) hist_add2(cells, n[a][e], now[e], n[a][e + 1], now[e + 1]);
                } else {
                    *reinterpret_cast<float*>(cells + n[a][0]) += now[0];
                }
                if constexpr (AXES > 1) wave_order();       // the halves change axes
            }
        }
    }
    __syncthreads();
    const int wave = tid >> 6, lane = tid & 63;
    const int64_t part = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, parts = (int64_t)gridDim.x * gridDim.y;
    for (int n = wave; n < nrows; n += BLOCK / 64) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < COLS / 64; ++k) s += hist[n * COLS + k * 64 + lane];
        s = wave_sum(s);
        if (lane == 0) partial[(h * parts + part) * nrows + n] = s;
    }
}

// joins `parts` partial tables of head blockIdx.y: gtable[row][h], row = a * buckets + n = blockIdx.x; one wave
__global__ __launch_bounds__(64) void rel_bias_join_kernel(const float* __restrict__ partial, void* __restrict__ gtable, int type,
                                                                 int H, int nrows, int64_t parts) {
    const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x;
    const float* p = partial + h * parts * nrows + row;
    double s = 0.0;
    for (int64_t i = lane; i < parts; i += 64) s += (double)p[i * nrows];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) {
        const int64_t at = (int64_t)row * H + h;
        if (type == CAMLI_F32) static_cast<float*>(gtable)[at] = (float)s;
        else if (type == CAMLI_BF16) static_cast<__bf16*>(gtable)[at] = (__bf16)(float)s;
        else static_cast<_Float16*>(gtable)[at] = (_Float16)(float)s;
    }
}

// does d^steps >= limit^j e^(steps - j) hold, exactly: both sides are products of `steps` factors below 2^11 (at most 704 bits)
bool reaches(int d, int limit, int e, int j, int steps) {
    uint32_t lhs[24] = {1}, rhs[24] = {1};
    auto mul = [](uint32_t* x, uint32_t f) {
        uint64_t carry = 0;
        for (int k = 0; k < 24; ++k) {
            carry += (uint64_t)x[k] * f;
            x[k] = (uint32_t)carry;
            carry >>= 32;
        }
    };
    for (int k = 0; k < steps; ++k) {
        mul(lhs, (uint32_t)d);
        mul(rhs, (uint32_t)(k < j ? limit : e));
    }
    for (int k = 23; k >= 0; --k)
        if (lhs[k] != rhs[k]) return lhs[k] > rhs[k];
    return true;
}

}  // namespace

bool rel_bias_args(RelBias& r, const char* who, const void* table, int type, const int* qpos, int64_t qpos_bs, const int* kpos,
                   int64_t kpos_bs, int axes, int buckets, int two_sided, int limit) {
    const int side = two_sided ? buckets / 2 : buckets, exact = side / 2;
    if (!table || !qpos || !kpos || type < 0 || type > 2 || axes < 1 || axes > 2 || (two_sided && buckets % 2 != 0) || side < 2 ||
        axes * buckets > CAMLI_REL_MAX_ROWS || limit > CAMLI_REL_MAX_LIMIT || limit <= exact) {
        camli_set_error("%s: position bias needs a table, positions, 1 or 2 axes, at least 2 buckets a side (an even number of buckets when two-sided), axes * buckets <= %d, buckets a side / 2 < max_distance <= %d "
                        "(axes=%d buckets=%d two_sided=%d max_distance=%d type=%d)", who, CAMLI_REL_MAX_ROWS, CAMLI_REL_MAX_LIMIT, axes, buckets, two_sided, limit, type);
        return false;
    }
    r.table = table; r.type = type; r.qpos = qpos; r.kpos = kpos; r.qpos_bs = qpos_bs; r.kpos_bs = kpos_bs;
    r.axes = axes; r.buckets = buckets; r.side = side; r.exact = exact; r.two_sided = two_sided ? 1 : 0; r.limit = limit;
    const int steps = side - exact;
    r.n_borders = steps - 1;
    for (int j = 1; j < steps; ++j) {
        // the logarithm places the border; within 1e-6 of a whole number the integers decide
        const double t = exact * pow((double)limit / exact, (double)j / steps);
        const double near = floor(t + 0.5);
        int d = (int)ceil(t);
        if (fabs(t - near) < 1e-6) d = reaches((int)near, limit, exact, j, steps) ? (int)near : (int)near + 1;
        r.border[j - 1] = d;
    }
    for (int j = r.n_borders; j < CAMLI_REL_MAX_BORDERS; ++j) r.border[j] = INT32_MAX;
    return true;
}

int rel_bias_join(const float* partial, void* gtable, int type, int H, int nrows, int64_t parts, const char* who, hipStream_t s) {
    rel_bias_join_kernel<<<dim3(nrows, H), 64, 0, s>>>(partial, gtable, type, H, nrows, parts);
    return camli_check_launch(who);
}

namespace {

int pow2_cols(int n) {      // threads along a row: the power of two that covers it, at most a workgroup
    int c = 1;
    while (c < n && c < BLOCK) c *= 2;
    return c;
}

size_t bwd_lds(int axes, int buckets, int limit) { return sizeof(float) * axes * buckets * bwd_columns(axes) + 2 * (2 * limit + 2); }

// row parts per column tile: as many workgroups as fit on the chip at once (two to four a CU), but 16 row groups in each: a workgroup pays for its table
// and for clearing and adding up its histogram
int bwd_parts(int64_t rows, int Lk, int H, int vec, int axes, int buckets) {
    const int fit = (int)((size_t)159 * 1024 / bwd_lds(axes, buckets, CAMLI_REL_MAX_LIMIT));
    const int64_t want = 256 * (fit < 2 ? 2 : fit > 4 ? 4 : fit);
    const int cols = pow2_cols(camli_divup(Lk, vec)), per = BLOCK / cols, tiles = camli_divup(Lk, cols * vec);
    const int64_t most = (want + (int64_t)H * tiles - 1) / ((int64_t)H * tiles), few = ((rows + per - 1) / per + 15) / 16;
    return (int)(few < most ? few : most);
}

template <typename T, int VEC, int AXES>
int fwd(const RelBias& r, void* out, int B, int H, int Lq, int Lk, hipStream_t s) {
    const int cols = pow2_cols(camli_divup(Lk, VEC)), per = BLOCK / cols;
    const dim3 grid(camli_divup(Lk, cols * VEC), camli_divup(Lq, ROWS * per), B * H);
    rel_bias_fwd_kernel<T, VEC, AXES><<<grid, BLOCK, sizeof(float) * AXES * (2 * r.limit + 1), s>>>(r, static_cast<T*>(out), H, Lq, Lk, cols);
    return camli_check_launch("camli_rel_bias_fwd");
}

template <typename T, int VEC, int AXES>
int bwd(const RelBias& r, const void* g, void* gtable, float* ws, int B, int H, int Lq, int Lk, hipStream_t s) {
    static unsigned long long done = 0;
    if (!camli_reserve_lds((const void*)rel_bias_bwd_kernel<T, VEC, AXES>, bwd_lds(1, CAMLI_REL_MAX_ROWS, CAMLI_REL_MAX_LIMIT), done)) {
        camli_set_error("camli_rel_bias_bwd: cannot reserve LDS");
        return CAMLI_ELAUNCH;
    }
    const int64_t rows = (int64_t)B * Lq;
    const int nrows = AXES * r.buckets, cols = pow2_cols(camli_divup(Lk, VEC)), parts = bwd_parts(rows, Lk, H, VEC, AXES, r.buckets);
    const int tiles = camli_divup(Lk, cols * VEC);
    const size_t lds = bwd_lds(AXES, r.buckets, r.limit);
    rel_bias_bwd_kernel<T, VEC, AXES><<<dim3(parts, tiles, H), BLOCK, lds, s>>>(r, static_cast<const T*>(g), ws, H, Lq, Lk, rows, cols);
    return rel_bias_join(ws, gtable, r.type, H, nrows, (int64_t)parts * tiles, "camli_rel_bias_bwd", s);
}

bool sizes_ok(int B, int H, int Lq, int Lk, const char* who) {
    if (B < 1 || H < 1 || Lq < 1 || Lk < 1 || (int64_t)B * H > 65535 || Lq > 2000000 || Lk > 16000000) {
        camli_set_error("%s: need B, H, Lq, Lk >= 1, B * H <= 65535, Lq <= 2000000, Lk <= 16000000 (B=%d H=%d Lq=%d Lk=%d)", who, B, H, Lq, Lk);
        return false;
    }
    return true;
}

template <typename T>
int fwd_any(const RelBias& r, void* out, int B, int H, int Lq, int Lk, hipStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = Lk % VEC == 0 && ((uintptr_t)out & 15) == 0;
    if (r.axes == 1) return vec ? fwd<T, VEC, 1>(r, out, B, H, Lq, Lk, s) : fwd<T, 1, 1>(r, out, B, H, Lq, Lk, s);
    return vec ? fwd<T, VEC, 2>(r, out, B, H, Lq, Lk, s) : fwd<T, 1, 2>(r, out, B, H, Lq, Lk, s);
}

template <typename T>
int bwd_any(const RelBias& r, const void* g, void* gt, float* ws, int B, int H, int Lq, int Lk, hipStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = Lk % VEC == 0 && ((uintptr_t)g & 15) == 0;
    if (r.axes == 1) return vec ? bwd<T, VEC, 1>(r, g, gt, ws, B, H, Lq, Lk, s) : bwd<T, 1, 1>(r, g, gt, ws, B, H, Lq, Lk, s);
    return vec ? bwd<T, VEC, 2>(r, g, gt, ws, B, H, Lq, Lk, s) : bwd<T, 1, 2>(r, g, gt, ws, B, H, Lq, Lk, s);
}

}  // namespace

extern "C" int camli_rel_bias_borders(int buckets, int two_sided, int max_distance, int* border) {
    RelBias r;
    const int dummy = 0;
    if (!border || !rel_bias_args(r, "camli_rel_bias_borders", &dummy, 0, &dummy, 0, &dummy, 0, 1, buckets, two_sided, max_distance)) return CAMLI_EINVAL;
    for (int j = 0; j < r.n_borders; ++j) border[j] = r.border[j];
    return r.n_borders;
}

extern "C" int camli_rel_bias_fwd(const void* table, const int* q_pos, int64_t q_pos_batch_stride, const int* k_pos, int64_t k_pos_batch_stride,
                                  void* out, int B, int H, int Lq, int Lk, int axes, int buckets, int two_sided, int max_distance, int type,
                                  void* stream) {
    RelBias r;
    if (!sizes_ok(B, H, Lq, Lk, "camli_rel_bias_fwd") ||
        !rel_bias_args(r, "camli_rel_bias_fwd", table, type, q_pos, q_pos_batch_stride, k_pos, k_pos_batch_stride, axes, buckets, two_sided, max_distance))
        return CAMLI_EINVAL;
    if (!out) { camli_set_error("camli_rel_bias_fwd: null output"); return CAMLI_EINVAL; }
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (type == CAMLI_F32) return fwd_any<float>(r, out, B, H, Lq, Lk, s);
    if (type == CAMLI_BF16) return fwd_any<__bf16>(r, out, B, H, Lq, Lk, s);
    return fwd_any<_Float16>(r, out, B, H, Lq, Lk, s);
}

extern "C" int64_t camli_rel_bias_bwd_workspace_bytes(int B, int H, int Lq, int Lk, int axes, int buckets, int type) {
    if (!sizes_ok(B, H, Lq, Lk, "camli_rel_bias_bwd_workspace_bytes") || axes < 1 || axes > 2 || buckets < 1 || type < 0 || type > 2) return 0;
    const int vec = 16 / camli_type_size(type);
    const int64_t rows = (int64_t)B * Lq;
    // whichever form the alignment allows
    const int64_t a = (int64_t)bwd_parts(rows, Lk, H, vec, axes, buckets) * camli_divup(Lk, pow2_cols(camli_divup(Lk, vec)) * vec);
    const int64_t c = (int64_t)bwd_parts(rows, Lk, H, 1, axes, buckets) * camli_divup(Lk, pow2_cols(Lk));
    return (int64_t)sizeof(float) * H * (a > c ? a : c) * axes * buckets;
}

extern "C" int camli_rel_bias_bwd(const void* gout, const int* q_pos, int64_t q_pos_batch_stride, const int* k_pos, int64_t k_pos_batch_stride,
                                  void* gtable, void* workspace, int64_t workspace_bytes, int B, int H, int Lq, int Lk, int axes, int buckets,
                                  int two_sided, int max_distance, int type, void* stream) {
    RelBias r;
    if (!sizes_ok(B, H, Lq, Lk, "camli_rel_bias_bwd") ||
        !rel_bias_args(r, "camli_rel_bias_bwd", gtable, type, q_pos, q_pos_batch_stride, k_pos, k_pos_batch_stride, axes, buckets, two_sided, max_distance))
        return CAMLI_EINVAL;
    if (!gout || !workspace || workspace_bytes < camli_rel_bias_bwd_workspace_bytes(B, H, Lq, Lk, axes, buckets, type)) {
        camli_set_error("camli_rel_bias_bwd: null pointer or workspace too small");
        return CAMLI_EINVAL;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* ws = static_cast<float*>(workspace);
    if (type == CAMLI_F32) return bwd_any<float>(r, gout, gtable, ws, B, H, Lq, Lk, s);
    if (type == CAMLI_BF16) return bwd_any<__bf16>(r, gout, gtable, ws, B, H, Lq, Lk, s);
    return bwd_any<_Float16>(r, gout, gtable, ws, B, H, Lq, Lk, s);
}
