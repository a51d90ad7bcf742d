// Learned relative position bias by buckets: what relbias.hip and the attention kernels (xattn.h) share.
//
//   bias[h, i, j] = sum_a table[a, bucket(kpos[j, a] - qpos[i, a]), h],    a = 0 .. axes - 1
//
// bucket(o), two-sided: side = buckets / 2, d = |o|, + side where o > 0; one-sided: side = buckets, d = max(-o, 0).  Distances
// below e = side / 2 have a bucket each; beyond, bucket e + j starts at the smallest d with d >= e (limit / e)^(j / (side - e)), and
// the last one has no end.  The borders are whole numbers found on the host in exact arithmetic (rel_bias_borders); they travel as
// kernel arguments, so no call uploads anything and a captured graph holds everything it needs.
//
// Offsets beyond +-limit share the bucket of the limit: a workgroup expands its heads' table columns to one float per offset in
// LDS (2 limit + 1 entries).
#pragma once
#include "typed.h"

#define CAMLI_REL_MAX_LIMIT 1023
#define CAMLI_REL_MAX_ROWS 128      // axes * buckets
#define CAMLI_REL_MAX_BORDERS 64

struct RelBias {
    const void* table;          // [axes][buckets][H]
    const int *qpos, *kpos;     // [.., L, axes], batch strides in ints (0: shared)
    int64_t qpos_bs, kpos_bs;
    int type, axes, buckets, side, exact, two_sided, limit, n_borders;
    int border[CAMLI_REL_MAX_BORDERS];      // INT_MAX from n_borders on
};

// fills r; false (with the error set) for arguments outside the documented range
bool rel_bias_args(RelBias& r, const char* who, const void* table, int type, const int* qpos, int64_t qpos_bs, const int* kpos,
                   int64_t kpos_bs, int axes, int buckets, int two_sided, int limit);

// gtable[row][h] = sum over parts of partial[h][part][row], row = a * buckets + n, in a fixed order and in 64 bits
int rel_bias_join(const float* partial, void* gtable, int type, int H, int nrows, int64_t parts, const char* who, hipStream_t s);

// The borders in LDS, for rel_bucket (kernel arguments with a lane's own index are memory reads, and all 64 in scalar registers displace
// what the callers' loops need).  Called by all threads; ends with a barrier.
__device__ __forceinline__ const int* rel_stage_borders(const RelBias& r) {
    __shared__ int border[CAMLI_REL_MAX_BORDERS];
    if (threadIdx.x < CAMLI_REL_MAX_BORDERS) border[threadIdx.x] = r.border[threadIdx.x];
    __syncthreads();
    return border;
}

// bucket of the clamped offset index i in 0 .. 2 limit
__device__ __forceinline__ int rel_bucket(const RelBias& r, const int* border, int i) {
    const int o = i - r.limit;
    const int d = r.two_sided ? abs(o) : max(-o, 0);
    int n = d;
    if (d >= r.exact) {
        int below = 0;          // borders at or below d, by bisection: at most 63 are in use, the others are INT_MAX
#pragma unroll
        for (int step = CAMLI_REL_MAX_BORDERS / 2; step >= 1; step >>= 1) below += border[below + step - 1] <= d ? step : 0;
        n = r.exact + below;
    }
    return n + (r.two_sided && o > 0 ? r.side : 0);
}

// A pair's table entry in LDS by one addition and one clamp.  Positions are held as multiples of the entry size (scaled once per row, not
// per pair), one side negated and carrying the address of the table's middle.  Positions beyond +-2^26 count as that, so that no
// difference overflows.
__device__ __forceinline__ unsigned lds_address(const void* p) {
    return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
template <typename V>
__device__ __forceinline__ V lds_load(int address) {
    return *(__attribute__((address_space(3))) const V*)(uintptr_t)(unsigned)address;
}
__device__ __forceinline__ int med3(int x, int lo, int hi) {
    int r;
    asm("v_med3_i32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(lo), "v"(hi));
    return r;
}
template <int SCALE>
__device__ __forceinline__ int scale_pos(int pos) { return min(max(pos, -(1 << 26)), 1 << 26) * SCALE; }

// orders a wave's LDS accesses (they execute in order; this keeps the compiler from moving them)
__device__ __forceinline__ void wave_order() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Two additions to a column of a histogram, at byte offsets.  Plain reads and writes: an LDS float add serialises its lanes here (193 cycles per
// wave instruction and CU measured, against 12 for a dependent read-add-write).  They may be, because no other thread writes these cells at
// the same time.  One axis: a column is one thread's.  Two: lanes l and l + 32 of a wave share a column and are among the rows of different
// axes at any time; wave_order() stands where they change axes.  The two cells may be the same one.
__device__ __forceinline__ void hist_add2(char* cells, unsigned at0, float v0, unsigned at1, float v1) {
    float x0 = *reinterpret_cast<float*>(cells + at0), x1 = *reinterpret_cast<float*>(cells + at1);
    x0 += v0;
    x1 = (at0 == at1 ? x0 : x1) + v1;
    *reinterpret_cast<float*>(cells + at0) = x0;
    *reinterpret_cast<float*>(cells + at1) = x1;
}
