// Cross attention over keys and values of another length, with an optional bucketed position bias: forward, both adjoints, gfx950.
// The instantiations are in files of their own, by kernel and element type (xattn_{fwd,dq,dkdv,far}_{f32,bf16,f16}.hip); checks, split rules
// and the C entries are in xattn.hip.
//
//   s_ij = scale q_i . k_j + bias[h, i, j],   p = softmax_j over the kept keys,   o_i = sum_j p_ij v_j      (no kept key: o_i = 0)
//   D_i = do_i . o_i,   dp_ij = do_i . v_j,   ds = p (dp - D),   dq = scale ds k,   dk = scale ds^T q,   dv = p^T do,
//   dtable[a, n, h] = sum of ds over the pairs whose bucket on axis a is n
//
// One scheme for all three kernels.  A wave OWNS 32 rows of one side (queries in fwd and dq, keys in dkdv) whose vectors sit in
// registers as the B operand of 32x32 matrix instructions, one row per lane (lanes l and l + 32 share row l); the other side streams
// through LDS in row-major tiles that all waves share.  The product tile then has the owned row on the lanes and the streamed rows in
// the 16 accumulator registers, so
//   * softmax statistics are per lane: no cross-lane traffic but one half-wave swap per tile,
//   * the same registers, rounded to the element type, ARE the B operand of the second product (the contraction order over the
//     streamed rows is free as long as both operands agree on it): P never leaves the registers,
//   * the A operand of the second product is the streamed tile transposed, read with the transposing LDS load.
// Register i of half h holds streamed row 8 (i / 4) + 4 h + i % 4 of its 32-row block.
//
// fp16 dS: p (dp - D) is of the size of |go| |v| / Lk, for ordinary operands below fp16's normal numbers, for large values beyond its largest.
// |dp - D| is at most 2 |go|_1 max|v| (out is a mean of values), so dS is taken times the power of two that brings this bound to 2^14 .. 2^15: it
// cannot overflow, and what it loses is below 2^-39 of the bound.  max|v| is over the kept keys of a kv head (a launch before the others), |go|_1 a
// row's own in dq, where the contraction is over keys, and the largest of the kv head in dkdv, where it is over queries.  In dq go itself is
// an operand: it is taken times a power of two that brings its largest element to 1 .. 2, and p times what is left.  P is taken times 2^10 in
// dkdv.  All of these are undone exactly when the gradients are written.
//
// Two adjoint kernels recompute p instead of one that adds dq with float atomics: 14 D instead of 10 D operations per pair, but
// every sum has a fixed order (the same bits on every run).  P and dS are rounded to the element type for the second products (their
// sums stay fp32): half a step of the inputs' own type, as for every operand of a matrix product.
#pragma once
#include "camli_hip.h"
#include "relbias.h"

namespace xattn {

struct Strides {
    int64_t b, l, h;            // elements
};

struct Args {
    const void *q, *k, *v, *go;
    const float *o;
    Strides qs, ks, vs;         // o, go and the gradients are dense [B][L][heads][D]
    void *out, *dq, *dk, *dv;
    float *out_f32;             // 16-bit types in training: out before its rounding
    float* lse;                 // [2][B][H][Lq], log2 domain, two terms; +inf where no key is kept
    float *delta;               // [B][H][Lq]
    float* go_l1;               // [B][H][Lq] fp16 only: sum of |go| of a row
    float* v_max;               // [B][Hk][v_chunks] fp16 only: largest |v| of a chunk of the kept keys
    int *far_rows;              // [B][H][row_groups]: has any of 32 queries a far lse
    float *part_o, *part_lse;   // splits > 1: [split][B][Lq][H][D] normalised, [2][split][B][H][Lq] (two terms, -inf: no key)
    float *part_dk, *part_dv;   // splits > 1: [split][B][Lk][Hk][D]
    float *part_table;          // [H][parts][axes * buckets]
    const int *lengths;         // [B] or null
    const unsigned char *mask;  // [B][mask_bs] or null
    int64_t mask_bs;
    int B, H, Hk, Lq, Lk, D;
    bool few;                   // fwd_few_kernel
    int pack;                   // query heads of one kv head that share a workgroup's rows (few queries), else 1
    int row_tiles, splits, tiles_per_split, parts, row_groups, v_chunks;
    float scale, scale_log2;
    RelBias rb;
};

typedef float acc16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef unsigned uint2v __attribute__((ext_vector_type(2)));
typedef unsigned chunk16 __attribute__((ext_vector_type(4)));       // 16 bytes in flight

// 16-byte fragments: what a lane holds of one operand for one k-step
template <typename L> struct Mat;
template <> struct Mat<__bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ acc16 mma(frag a, frag b, acc16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mat<_Float16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ acc16 mma(frag a, frag b, acc16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

// fp32 operands are held as three bf16 parts, x = x0 + x1 + x2 exactly (each the rounding of what is left: 8 + 8 + 8 bits), and a product
// is the six terms a0 b0, a0 b1, a1 b0, a1 b1, a0 b2, a2 b0 in fp32 accumulators, smallest first.  What is left out, a1 b2 + a2 b1 + a2 b2,
// is at most 2^-25 of |a| |b|: less than fp32's own rounding of the product.  A 32 x 32 x 32 product takes 384 cycles of the matrix
// unit so, 1024 as fp32 instructions (2 x 2048 queries x 8160 keys x 4 heads of 32 with a two-axis bias, forward and backward: 854 -> 588 us;
// heads of 128 without one: 2650 -> 1730 us).  (An infinity has no parts: it comes out as NaN.)
template <typename T> struct Parts {
    typedef T Lds;
    static constexpr int N = 1;
};
template <> struct Parts<float> {
    typedef __bf16 Lds;
    static constexpr int N = 3;
};

template <int I>
struct Int {
    static constexpr int value = I;
};

template <typename T>
struct Frag {
    typename Mat<typename Parts<T>::Lds>::frag part[Parts<T>::N];
};

template <typename T>
__device__ __forceinline__ acc16 mma(const Frag<T>& a, const Frag<T>& b, acc16 c) {
    using M = Mat<typename Parts<T>::Lds>;
    if constexpr (Parts<T>::N == 3) {
        c = M::mma(a.part[2], b.part[0], c);
        c = M::mma(a.part[0], b.part[2], c);
        c = M::mma(a.part[1], b.part[1], c);
        c = M::mma(a.part[1], b.part[0], c);
        c = M::mma(a.part[0], b.part[1], c);
    }
    return M::mma(a.part[0], b.part[0], c);
}

typedef float float2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// 8 floats -> the parts of type T (in pairs: one conversion instruction rounds two)
template <typename T>
__device__ __forceinline__ Frag<T> to_frag(const float (&x)[8]) {
    typedef typename Parts<T>::Lds L;
    typedef L pair __attribute__((ext_vector_type(2)));
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float2v v = {x[i], x[i + 1]};
#pragma unroll
        for (int n = 0; n < Parts<T>::N; ++n) {
            const pair r = __builtin_convertvector(v, pair);
            f.part[n][i] = r[0];
            f.part[n][i + 1] = r[1];
            v[0] -= (float)r[0];
            v[1] -= (float)r[1];
        }
    }
    return f;
}

// A tile of R streamed rows in LDS, one plane per part.  Rows are unpadded and their 16-byte chunks permuted by an XOR with bits of the row,
// chosen so that both readers hit every bank equally: 16 lanes reading one chunk of 16 rows, and the transposing load's 8 rows x 64 bytes.
template <typename T, int DP, int R>
struct Tile {
    using Lds = typename Parts<T>::Lds;
    static constexpr int E = 8;                         // elements of a 16-byte chunk
    static constexpr int CHUNKS = DP / E;               // chunks of a row
    static constexpr int ROWS = R;
    static constexpr int BLOCKS = ROWS / 32;
    static constexpr int PLANE = ROWS * DP;
    static constexpr int ELEMS = Parts<T>::N * PLANE;
    static constexpr int KSTEPS = CHUNKS / 2;           // k-steps of a product over DP
    static constexpr int PSTEPS = 2;                    // k-steps of a product over 32 streamed rows
    static constexpr int DBLOCKS = DP / 32;

    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (CHUNKS == 4) return (row >> 2) & 3;
        else if constexpr (CHUNKS == 8) return ((row >> 1) & 1) << 2 | ((row >> 2) & 3);
        else return (row & 7) << 1 | ((row >> 3) & 1);
    }
    static __device__ __forceinline__ int chunk_at(int row, int c) { return row * DP + (c ^ swizzle(row)) * E; }
};

// rows of a streamed tile: what a thread of 256 can fetch at once in narrow heads, what two buffers leave room for in wide fp32 ones
constexpr int tile_rows(int size, int dp) { return size == 2 || dp == 32 ? 64 : 32; }
// dq with a histogram beside one buffer: small tiles leave LDS for three workgroups a CU in narrow heads (64 rows: 1089 us where 32 take 1063)
constexpr int dq_tile_rows(int size, int dp, bool hist) { return hist ? 32 : tile_rows(size, dp); }

// Where a lane reads in a tile (element offsets from the start of a 32-row block; loop-invariant).
template <typename TL, typename T>
struct LaneMap {
    using L = typename TL::Lds;
    int row[TL::KSTEPS];                                        // A operand of products over DP: row lane % 32, chunk 2 s + half
    int col[TL::DBLOCKS][2];                                    // A operand of products over the streamed rows

    __device__ __forceinline__ explicit LaneMap(int lane) {
        const int h = lane >> 5, l = lane & 15;
#pragma unroll
        for (int s = 0; s < TL::KSTEPS; ++s) row[s] = TL::chunk_at(lane & 31, 2 * s + h);
        // the transposing load: 16 lanes fetch 4 rows x 16 columns (8 bytes each) and receive a column's 4 rows each
#pragma unroll
        for (int d = 0; d < TL::DBLOCKS; ++d)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = d * 32 + (lane & 16) + (l & 3) * 4;
                col[d][u] = TL::chunk_at(4 * h + (l >> 2) + 8 * u, c / TL::E) + c % TL::E;
            }
    }
    __device__ __forceinline__ Frag<T> read_row(const L* block, int s) const {
        Frag<T> f;
#pragma unroll
        for (int n = 0; n < Parts<T>::N; ++n) f.part[n] = *reinterpret_cast<const typename Mat<L>::frag*>(block + n * TL::PLANE + row[s]);
        return f;
    }
    // column 32 d + lane % 32 of the rows of k-step t, in the order the accumulator has them
    __device__ __forceinline__ Frag<T> read_col(const L* block, int t, int d) const {
        typedef __attribute__((address_space(3))) short4v* lds_ptr;
        Frag<T> f;
#pragma unroll
        for (int n = 0; n < Parts<T>::N; ++n) {
            union { short4v s[2]; typename Mat<L>::frag f; } u;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                u.s[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(const_cast<L*>(block + n * TL::PLANE + 16 * t * 32 * TL::DBLOCKS + col[d][i])));
            f.part[n] = u.f;
        }
        return f;
    }
};

// c + block . own over DP
template <typename T, typename TL>
__device__ __forceinline__ acc16 product(const LaneMap<TL, T>& map, const typename TL::Lds* block, const Frag<T>* own, acc16 c) {
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks) c = mma<T>(map.read_row(block, ks), own[ks], c);
    return c;
}

// k-step t of the accumulator as an operand of type T
template <typename T>
__device__ __forceinline__ Frag<T> pack_step(const acc16& x, int t) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[t * 8 + i];
    return to_frag<T>(v);
}

// what that rounding left (16-bit types)
template <typename T>
__device__ __forceinline__ Frag<T> pack_rest(const acc16& x, const Frag<T>& rounded, int t) {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = x[t * 8 + i] - (float)rounded.part[0][i];
    return to_frag<T>(v);
}

__device__ __forceinline__ acc16 splat(float x) {
    acc16 v;
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = x;
    return v;
}

__device__ __forceinline__ int acc_row(int i, int h) { return (i >> 2) * 8 + 4 * h + (i & 3); }

__device__ __forceinline__ float other_half(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(threadIdx.x & 32 ? r[0] : r[1]);
}
__device__ __forceinline__ float half_max(float x) { return fmaxf(x, other_half(x)); }
__device__ __forceinline__ float half_sum(float x) { return x + other_half(x); }

// Workgroups go round-robin over the 8 XCDs.  The `chunk` workgroups of a unit (a sample's head: they stream the same keys and values, or
// queries) are kept on one XCD, so that they share its L2, and units alternate between the XCDs, so that samples of different lengths
// spread over them (contiguous ranges of samples per XCD took twice as long with lengths from 0 to 16384).
__device__ __forceinline__ int unit_per_xcd(int id, int n, int chunk) {
    const int units = n / chunk, full = (units >> 3) * 8 * chunk;
    int unit, k;
    if (id < full) {
        const int group = id / (8 * chunk), rem = id - group * 8 * chunk;
        unit = group * 8 + (rem & 7);
        k = rem >> 3;
    } else {
        const int left = units & 7, rem = id - full;
        unit = units - left + rem % left;
        k = rem / left;
    }
    return unit * chunk + k;
}

// 8 elements as they came from memory (one or two 16-byte loads) -> the parts of type T
template <typename T, int C>
__device__ __forceinline__ Frag<T> chunk_frag(const chunk16 (&v)[C]) {
    if constexpr (C == 1) {
        Frag<T> f;
        f.part[0] = __builtin_bit_cast(typename Mat<T>::frag, v[0]);
        return f;
    } else {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(v[i / 4][i % 4]);
        return to_frag<T>(x);
    }
}
// ... into a chunk of a tile, zeros if not kept
template <typename T, typename TL, int C>
__device__ __forceinline__ void put_chunk(typename TL::Lds* to, const chunk16 (&v)[C], bool kept) {
    using L = typename TL::Lds;
    chunk16 k[C];
#pragma unroll
    for (int i = 0; i < C; ++i) k[i] = kept ? v[i] : chunk16{0, 0, 0, 0};
    const Frag<T> parts = chunk_frag<T>(k);
#pragma unroll
    for (int n = 0; n < Parts<T>::N; ++n) *reinterpret_cast<typename Mat<L>::frag*>(to + n * TL::PLANE) = parts.part[n];
}
// The streamed pair of tiles on its way from memory: registers now, LDS later.  A row at or beyond `limit`, a masked row and columns
// from D on become zeros (a masked row may hold anything, and 0 * NaN is NaN); a whole, unmasked tile skips those tests.
// A thread's place in a tile is a 32-bit byte offset computed once (row strides are below 2^23 elements); the tile's base is uniform.
template <typename T, int DP, int R, int THREADS>
struct Stream {
    using TL = Tile<T, DP, R>;
    using L = typename TL::Lds;
    static constexpr int ALL = TL::ROWS * TL::CHUNKS, N = (ALL + THREADS - 1) / THREADS;      // the smallest tile has chunks for half the threads
    static constexpr int C = TL::E * sizeof(T) / 16;                                           // loads a chunk
    static_assert(ALL % THREADS == 0 || N == 1, "a whole number of chunks a thread");
    chunk16 x[N][C], y[N][C];
    unsigned at_x[N], at_y[N];
    unsigned keep;
    bool whole;

    __device__ __forceinline__ void init(int64_t ldx, int64_t ldy) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int f = threadIdx.x + n * THREADS;
            const unsigned c = (f % TL::CHUNKS) * 16 * C;
            at_x[n] = (unsigned)(f / TL::CHUNKS) * (unsigned)(ldx * (int)sizeof(T)) + c;
            at_y[n] = (unsigned)(f / TL::CHUNKS) * (unsigned)(ldy * (int)sizeof(T)) + c;
        }
    }
    // px, py: the tile's first row
    __device__ __forceinline__ void load(const T* px, const T* py, int row0, int limit, int D, const unsigned char* mask) {
        const char *bx = reinterpret_cast<const char*>(px), *by = reinterpret_cast<const char*>(py);
        whole = ALL >= THREADS && row0 + TL::ROWS <= limit && D == DP && mask == nullptr;
        if (whole) {
#pragma unroll
            for (int n = 0; n < N; ++n) fetch(n, bx, by);
            return;
        }
        keep = 0;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int f = threadIdx.x + n * THREADS, row = row0 + f / TL::CHUNKS, c = (f % TL::CHUNKS) * TL::E;
#pragma unroll
            for (int i = 0; i < C; ++i) x[n][i] = y[n][i] = chunk16{0, 0, 0, 0};
            if (row < limit && c < D && (ALL >= THREADS || f < ALL)) {
                fetch(n, bx, by);
                keep |= (mask == nullptr || mask[row] != 0 ? 1u : 0u) << n;
            }
        }
    }
    __device__ __forceinline__ void store(L* tx, L* ty) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int f = threadIdx.x + n * THREADS, at = TL::chunk_at(f / TL::CHUNKS, f % TL::CHUNKS);
            if (ALL < THREADS && f >= ALL) break;
            put_chunk<T, TL>(tx + at, x[n], whole || ((keep >> n) & 1));
            put_chunk<T, TL>(ty + at, y[n], whole || ((keep >> n) & 1));
        }
    }

private:
    __device__ __forceinline__ void fetch(int n, const char* bx, const char* by) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            x[n][i] = *reinterpret_cast<const chunk16*>(bx + at_x[n] + 16 * i);
            y[n][i] = *reinterpret_cast<const chunk16*>(by + at_y[n] + 16 * i);
        }
    }
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        load_f32<T, 8>(p, v);
    } else {
        float a[4], b[4];
        load_f32<T, 4>(p, a);
        load_f32<T, 4>(p + 4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
}

// The matrix unit aligns the terms of a sum to the largest and cuts what is below, downwards: every fp32 dp comes out 4e-8 (at |dp| of 6) too low,
// nothing to a gradient's element, but the bias table's gradient adds whole rows of ds that cancel and was off by 2e-5 of its size.  So every
// other owned row enters dp with its sign turned, and the shifts cancel.
template <typename T>
__device__ __forceinline__ float dp_sign(int lane) { return sizeof(T) == 4 && (lane & 1) ? -1.0f : 1.0f; }

// owned row, times sign (fp32) -> B fragments (zeros beyond D and for rows that do not exist)
template <typename T, int DP>
__device__ __forceinline__ void load_owned(Frag<T>* f, const T* row, bool exists, int D, int h, float sign = 1.0f) {
    using TL = Tile<T, DP, 32>;
#pragma unroll
    for (int s = 0; s < TL::KSTEPS; ++s) {
        const int c = (2 * s + h) * TL::E;
        f[s] = Frag<T>{};
        if (exists && c < D) {
            if constexpr (sizeof(T) == 2) {
                f[s].part[0] = *reinterpret_cast<const typename Mat<T>::frag*>(row + c);
            } else {
                float v[8];
                load8(row + c, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] *= sign;
                f[s] = to_frag<T>(v);
            }
        }
    }
}

// [DBLOCKS] accumulators (column of the owned row on the lane) -> dense row of elements, or of floats
template <typename O, int DBLOCKS>
__device__ __forceinline__ void store_owned(O* row, const acc16 (&o)[DBLOCKS], float mul, int D, int h) {
#pragma unroll
    for (int db = 0; db < DBLOCKS; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = db * 32 + acc_row(i, h);
            if (d < D) {
                const float v[4] = {o[db][i] * mul, o[db][i + 1] * mul, o[db][i + 2] * mul, o[db][i + 3] * mul};
                store_f32<O, 4>(row + d, v);
            }
        }
}

__device__ __forceinline__ int kept_length(const Args& a, int b) {
    return a.lengths ? min(max(a.lengths[b], 0), a.Lk) : a.Lk;
}

// bit j: key row0 + j is kept.  Called by whole waves.
__device__ __forceinline__ unsigned long long kept_bits(const unsigned char* mask, int row0, int len, int rows) {
    const unsigned long long all = rows == 64 ? ~0ull : (1ull << rows) - 1;
    if (mask == nullptr) return row0 + rows <= len ? all : (1ull << (len - row0)) - 1;      // row0 < len
    const int lane = threadIdx.x & 63, key = row0 + lane;
    bool k = lane < rows && key < len;
    if (k) k = mask[key] != 0;
    return __ballot(k);
}

// is streamed row acc_row(i, this lane's half) kept: the lanes' answers as a scalar mask, no vector instruction
__device__ __forceinline__ bool kept_row(unsigned kept, int i) {
    const int r = acc_row(i, 0);
    const unsigned lo = (unsigned)((int)(kept << (31 - r)) >> 31), hi = (unsigned)((int)(kept << (27 - r)) >> 31);
    return __builtin_amdgcn_inverse_ballot_w64((unsigned long long)hi << 32 | lo);
}

constexpr float LOG2E = 1.4426950408889634f;

// The bias of a pair comes from a table in LDS (rel_bias: relbias.h); query positions are the negated side.
// Entries: the bias (log2 domain), and for the table's gradient beside it where the bucket's row of the histogram starts.
struct Entry8 {
    float bias;
    unsigned hist;
};

// An entry of the table in the log2 domain.  Finite ones stay finite: the type's lowest number is a common mask, and log2 e times it is not a
// number, nor is the sum of two axes'.  At 2^125 such a sum and its distance from another one are.
__device__ __forceinline__ float lut_entry(const RelBias& r, int row, int H, int head) {
    const float x = load_param(r.table, r.type, (int64_t)row * H + head);
    return fabsf(x) < INFINITY ? fminf(fmaxf(x * LOG2E, -0x1p125f), 0x1p125f) : x;
}

// tables of `pack` heads: lut[p][axis][2 limit + 1]
template <int AXES, int THREADS>
__device__ __forceinline__ void fill_lut(const RelBias& r, float* lut, int head0, int pack, int H) {
    const int span = 2 * r.limit + 1;
    const int* border = rel_stage_borders(r);
    for (int i = threadIdx.x; i < span; i += THREADS) {
        const int n = rel_bucket(r, border, i);
        for (int p = 0; p < pack; ++p)
#pragma unroll
            for (int a = 0; a < AXES; ++a)
                lut[(p * AXES + a) * span + i] = lut_entry(r, a * r.buckets + n, H, head0 + p);
    }
}
template <int AXES, int THREADS>
__device__ __forceinline__ void fill_lut(const RelBias& r, Entry8* lut, int head, int row_bytes, int H) {
    const int span = 2 * r.limit + 1;
    const int* border = rel_stage_borders(r);
    for (int i = threadIdx.x; i < span; i += THREADS) {
        const int n = rel_bucket(r, border, i);
#pragma unroll
        for (int a = 0; a < AXES; ++a)
            lut[a * span + i] = {lut_entry(r, a * r.buckets + n, H, head), (unsigned)((a * r.buckets + n) * row_bytes)};
    }
}

// the same for lanes FIRST .. FIRST + 7
template <int FIRST>
__device__ __forceinline__ void broadcast_plus8(int lanes, int own, int (&out)[8]) {
    asm("s_nop 1\n\t"
        "v_add_u32_dpp %0, %8, %9 row_newbcast:%10 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %1, %8, %9 row_newbcast:%11 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %2, %8, %9 row_newbcast:%12 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %3, %8, %9 row_newbcast:%13 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %4, %8, %9 row_newbcast:%14 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %5, %8, %9 row_newbcast:%15 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %6, %8, %9 row_newbcast:%16 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %7, %8, %9 row_newbcast:%17 row_mask:0xf bank_mask:0xf"
        : "=&v"(out[0]), "=&v"(out[1]), "=&v"(out[2]), "=&v"(out[3]), "=&v"(out[4]), "=&v"(out[5]), "=&v"(out[6]), "=&v"(out[7])
        : "v"(lanes), "v"(own), "n"(FIRST + 0), "n"(FIRST + 1), "n"(FIRST + 2), "n"(FIRST + 3), "n"(FIRST + 4), "n"(FIRST + 5), "n"(FIRST + 6), "n"(FIRST + 7));
}

// bias of accumulator register i's pair: the axes' entries, added first (the order of two does not matter: every kernel gets the same bits)
template <int AXES>
__device__ __forceinline__ float pair_bias(const int (&off)[AXES][16], int i, const int (&lo)[AXES], const int (&hi)[AXES]) {
    float b = lds_load<float>(med3(off[0][i], lo[0], hi[0]));
    if constexpr (AXES > 1) b += lds_load<float>(med3(off[AXES - 1][i], lo[AXES - 1], hi[AXES - 1]));
    return b;
}

// Positions of the streamed rows stay out of LDS: lane i of each 16-lane row holds the position of the row that accumulator register i
// stands for (acc_row(i, h): the halves differ), and the subtraction reads it from there by a row broadcast.  As LDS broadcasts the
// same reads took a quarter of the LDS time.
template <int AXES, int BLOCKS, int SCALE>
struct StreamPos {
    int p[BLOCKS][AXES ? AXES : 1];

    // SWAP: the upper half takes the axes in the opposite order
    template <bool SWAP = false>
    __device__ __forceinline__ void load(const int* pos, int row0, int limit) {
        const int lane = threadIdx.x & 63, half = SWAP ? lane >> 5 : 0;
#pragma unroll
        for (int nb = 0; nb < BLOCKS; ++nb) {
            const int row = min(row0 + nb * 32 + acc_row(lane & 15, lane >> 5), limit - 1);
#pragma unroll
            for (int x = 0; x < AXES; ++x) p[nb][x] = scale_pos<SCALE>(pos[(int64_t)row * AXES + (x ^ half)]);
        }
    }
};
// out[i] = (lane i of the 16-lane row's `lanes`) + own.  One instruction each; the compiler does not fold this broadcast into the addition
// by itself.  (s_nop: a row broadcast may not read a register within two cycles of its writing.)
__device__ __forceinline__ void broadcast_plus(int lanes, int own, int (&out)[16]) {
    asm("s_nop 1\n\t"
        "v_add_u32_dpp %0, %16, %17 row_newbcast:0 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %1, %16, %17 row_newbcast:1 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %2, %16, %17 row_newbcast:2 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %3, %16, %17 row_newbcast:3 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %4, %16, %17 row_newbcast:4 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %5, %16, %17 row_newbcast:5 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %6, %16, %17 row_newbcast:6 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %7, %16, %17 row_newbcast:7 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %8, %16, %17 row_newbcast:8 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %9, %16, %17 row_newbcast:9 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %10, %16, %17 row_newbcast:10 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %11, %16, %17 row_newbcast:11 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %12, %16, %17 row_newbcast:12 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %13, %16, %17 row_newbcast:13 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %14, %16, %17 row_newbcast:14 row_mask:0xf bank_mask:0xf\n\t"
        "v_add_u32_dpp %15, %16, %17 row_newbcast:15 row_mask:0xf bank_mask:0xf"
        : "=&v"(out[0]), "=&v"(out[1]), "=&v"(out[2]), "=&v"(out[3]), "=&v"(out[4]), "=&v"(out[5]), "=&v"(out[6]), "=&v"(out[7]), "=&v"(out[8]), "=&v"(out[9]), "=&v"(out[10]), "=&v"(out[11]), "=&v"(out[12]), "=&v"(out[13]), "=&v"(out[14]), "=&v"(out[15])
        : "v"(lanes), "v"(own));
}

// ------------------------------------------------------------------------------------------------------------ references far from zero
// A finite table entry may be as low as its type goes, the usual mask of a bucket, and a row that so far has only such pairs (or no others
// at all) has its softmax reference there; products of large vectors get as far without a bias.  Next to such a number a float holds no
// digit of an ordinary score, so beyond FAR (log2 units; up to it a reference's own rounding is below 2^-16) nothing is computed
// relative to a reference before the reference is the tile's own, and a log-sum is two floats.
constexpr float FAR = 256.0f;

// a + b exactly, as hi + lo: lo is what the sum of a large a and a small b rounds away (0 within FAR; an infinity has none)
__device__ __forceinline__ void two_sum(float a, float b, float& hi, float& lo) {
    const float sum = a + b, bb = sum - a, rest = (a - (sum - bb)) + (b - bb);
    hi = sum;
    lo = fabsf(sum) > FAR && fabsf(sum) < INFINITY ? rest : 0.0f;
}
template <int N>
__device__ __forceinline__ void move_scores(acc16 (&s)[N], float by) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) s[n][i] += by;
}
__device__ __forceinline__ bool is_far(float lse) { return fabsf(lse) > FAR && lse < INFINITY; }      // +inf: a row without keys

// ------------------------------------------------------------------------------------------------------------ forward
// Softmax without a running maximum: the scores come out of the matrix unit already relative to m (the accumulators start at -m /
// scale; at zero while m is far), and m is taken from the first tile that has a kept key.  p <= 2^30 (2^14 for fp16) is as good as p <= 1 in floating point, so
// m moves only when a score passes that: the exchange between the half waves and the rescaling leave the loop, but for a test.
// TRAIN (16-bit types): out has to be known to more than its own type for the backward's D = do . o, which is subtracted from
// dp: P enters the product as two terms of the type and out is stored before its rounding as well.  Without that the bias table's
// gradient, a sum over whole rows of ds, is off by twice its own rounding.
// Measured: 4 x 8160 queries x 8160 keys, 2 heads of 128, bf16: 290 to 309 us from card to card, 880 to 940 TFLOP/s (a large library product: 1132), bound by the matrix
// unit; 8 x 8160 x 2048, 4 heads of 32 with a two-axis bias, bf16, training: 305 us, bound by vector arithmetic (14 instructions a pair, exp
// of four issue slots); the other way round in fp32, 2 x 2048 x 8160: 156 us.
// fp32 with a bias starts at zero and subtracts m at the end: at -m / scale every step of the product rounds to a few bits less (a relative
// error of p of 1e-6), which is nothing to a 16-bit product and shows in an fp32 gradient.  The adjoints do the same with the log-sum and D.
template <typename T>
constexpr bool fold_start() { return sizeof(T) == 2; }
template <typename T>
constexpr float exponent_limit() { return __is_same(T, _Float16) ? 14.0f : 30.0f; }

template <typename T, int DP, int AXES, bool TRAIN>
__global__ __launch_bounds__(256, DP == 32 ? (AXES || sizeof(T) == 4 ? 3 : 4) : DP == 64 || (sizeof(T) == 2 && AXES == 0) ? 2 : 1) void fwd_kernel(Args a) {
    constexpr int R = tile_rows(sizeof(T), DP);
    using TL = Tile<T, DP, R>;
    using L = typename TL::Lds;
    constexpr int THREADS = 256, ENTRY = (int)sizeof(float);
    constexpr bool TWO_TERMS = TRAIN && sizeof(T) == 2, FOLD = AXES > 0 && fold_start<T>();
    constexpr unsigned long long ALL_KEPT = R == 64 ? ~0ull : (1ull << R) - 1;
    extern __shared__ __align__(16) char smem[];
    L* tiles = reinterpret_cast<L*>(smem);                                  // [2][K, V]
    float* lut = reinterpret_cast<float*>(tiles + 4 * TL::ELEMS);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int id = unit_per_xcd(blockIdx.x, gridDim.x, a.row_tiles * a.splits);
    const int groups = a.H / a.pack;
    const int split = id % a.splits;
    id /= a.splits;
    const int rt = id % a.row_tiles;
    id /= a.row_tiles;
    const int hh = id % groups, b = id / groups, kvh = hh * a.pack / (a.H / a.Hk);
    const int row = rt * 128 + wave * 32 + (lane & 31), rows = a.pack * a.Lq;
    const bool exists = row < rows, busy = rt * 128 + wave * 32 < rows;         // an idle wave only helps to fetch
    const int sub = exists ? row / a.Lq : 0, qi = exists ? row - sub * a.Lq : 0, head = hh * a.pack + sub;

    const int len = kept_length(a, b);
    const int n_tiles = (len + TL::ROWS - 1) / TL::ROWS;
    const int t0 = split * a.tiles_per_split, t1 = min(n_tiles, t0 + a.tiles_per_split);
    const T* kp = static_cast<const T*>(a.k) + b * a.ks.b + kvh * a.ks.h;
    const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + kvh * a.vs.h;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_bs : nullptr;

    Frag<T> qf[TL::KSTEPS];
    load_owned<T, DP>(qf, static_cast<const T*>(a.q) + b * a.qs.b + qi * a.qs.l + head * a.qs.h, exists, a.D, h);
    int qa[AXES ? AXES : 1], lo[AXES ? AXES : 1], hi[AXES ? AXES : 1];
    const int* kpos = nullptr;
    if constexpr (AXES > 0) {
        fill_lut<AXES, THREADS>(a.rb, lut, hh * a.pack, a.pack, a.H);
        kpos = a.rb.kpos + b * a.rb.kpos_bs;
#pragma unroll
        for (int x = 0; x < AXES; ++x) {
            const int centre = (int)lds_address(lut + (sub * AXES + x) * (2 * a.rb.limit + 1) + a.rb.limit);
            qa[x] = centre + scale_pos<-ENTRY>(a.rb.qpos[b * a.rb.qpos_bs + (int64_t)qi * AXES + x]);
            lo[x] = centre - 4 * a.rb.limit;
            hi[x] = centre + 4 * a.rb.limit;
        }
    }
    const LaneMap<TL, T> map(lane);

    acc16 o[TL::DBLOCKS];
#pragma unroll
    for (int d = 0; d < TL::DBLOCKS; ++d) o[d] = acc16{0};
    // m: the reference of the row's exponents, log2 domain (-inf: no kept key yet, use 0); start: -m / scale in every accumulator (FOLD:
    // with a bias, unless any of the wave's rows is far; without one the exponent's multiply-add subtracts m at no cost)
    float m = -INFINITY, m_use = 0.0f, l = 0.0f;
    acc16 start = splat(0.0f);
    bool unset = true, far = false;

    Stream<T, DP, R, THREADS> st;
    StreamPos<AXES, TL::BLOCKS, ENTRY> pos, pos_next;
    st.init(a.ks.l, a.vs.l);
    int cur = 0;
    if (t0 < t1) {
        st.load(kp + t0 * (int64_t)TL::ROWS * a.ks.l, vp + t0 * (int64_t)TL::ROWS * a.vs.l, t0 * TL::ROWS, len, a.D, mask);
        if constexpr (AXES > 0) pos_next.load(kpos, t0 * TL::ROWS, len);
        st.store(tiles, tiles + TL::ELEMS);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const unsigned long long bits = kept_bits(mask, t * TL::ROWS, len, TL::ROWS);
        if constexpr (AXES > 0) pos = pos_next;
        if (t + 1 < t1) {
            st.load(kp + (t + 1) * (int64_t)TL::ROWS * a.ks.l, vp + (t + 1) * (int64_t)TL::ROWS * a.vs.l, (t + 1) * TL::ROWS, len, a.D, mask);
            if constexpr (AXES > 0) pos_next.load(kpos, (t + 1) * TL::ROWS, len);
        }
        const L *kt = tiles + cur * 2 * TL::ELEMS, *vt = kt + TL::ELEMS;
        if (bits != 0 && busy) {
            acc16 s[TL::BLOCKS];
            float top = -INFINITY;
#pragma unroll
            for (int nb = 0; nb < TL::BLOCKS; ++nb) {
                s[nb] = product<T, TL>(map, kt + nb * 32 * DP, qf, FOLD ? start : acc16{0});
            }
            if constexpr (AXES > 0) {
#pragma unroll
                for (int nb = 0; nb < TL::BLOCKS; ++nb) {
                    int off[AXES][16];
#pragma unroll
                    for (int x = 0; x < AXES; ++x) broadcast_plus(pos.p[nb][x], qa[x], off[x]);
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        s[nb][i] = __builtin_fmaf(s[nb][i], a.scale_log2, pair_bias<AXES>(off, i, lo, hi));
                    }
                }
            }
            if (bits != ALL_KEPT) {
#pragma unroll
                for (int nb = 0; nb < TL::BLOCKS; ++nb) {
                    const unsigned mine = (unsigned)(bits >> (nb * 32)) >> (4 * h);
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[nb][i] = (mine >> acc_row(i, 0)) & 1 ? s[nb][i] : -INFINITY;
                }
            }
#pragma unroll
            for (int nb = 0; nb < TL::BLOCKS; ++nb)
#pragma unroll
                for (int i = 0; i < 16; ++i) top = fmaxf(top, s[nb][i]);
            // base: what the scores are relative to.  Without a bias they are products still; the highest is rounded as the reference is, so
            // that it comes out as 0 next to any reference
            float base = FOLD && !far ? m_use : 0.0f;
            if constexpr (AXES == 0) top *= a.scale_log2;
            if (unset || __any(top + (base - m_use) > exponent_limit<T>())) {
                // a row's own need decides where its reference goes; rows beside it (far ones) change no more than when it is subtracted
                top = half_max(top);
                const float mn = m == -INFINITY || top + (base - m_use) > exponent_limit<T>() ? fmaxf(m, top + base) : m, use = mn == -INFINITY ? 0.0f : mn;
                const float alpha = __builtin_amdgcn_exp2f(m - use);
#pragma unroll
                for (int d = 0; d < TL::DBLOCKS; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
                l *= alpha;
                m = mn;
                m_use = use;
                unset = __any(m == -INFINITY);
                far = __any(fabsf(m_use) > FAR);
                if constexpr (FOLD) {
                    start = splat(far ? 0.0f : -use / a.scale_log2);
                    move_scores(s, base - use);
                }
            } else if (FOLD && far) {
                move_scores(s, -m_use);
            }
            const float mul = far ? 1.0f : a.scale_log2;
            if (AXES == 0 && far) {
#pragma unroll
                for (int nb = 0; nb < TL::BLOCKS; ++nb)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[nb][i] *= a.scale_log2;
            }
#pragma unroll
            for (int nb = 0; nb < TL::BLOCKS; ++nb) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    s[nb][i] = __builtin_amdgcn_exp2f(FOLD ? s[nb][i] : AXES > 0 ? s[nb][i] - m_use : __builtin_fmaf(s[nb][i], mul, -m_use));
                    l += s[nb][i];
                }
#pragma unroll
                for (int ps = 0; ps < TL::PSTEPS; ++ps) {
                    const Frag<T> p = pack_step<T>(s[nb], ps);
                    Frag<T> rest;
                    if constexpr (TWO_TERMS) rest = pack_rest<T>(s[nb], p, ps);
#pragma unroll
                    for (int d = 0; d < TL::DBLOCKS; ++d) {
                        const Frag<T> v = map.read_col(vt + nb * 32 * DP, ps, d);
                        o[d] = mma<T>(v, p, o[d]);
                        if constexpr (TWO_TERMS) o[d] = mma<T>(v, rest, o[d]);
                    }
                }
            }
        }
        if (t + 1 < t1) {
            L* nk = tiles + (cur ^ 1) * 2 * TL::ELEMS;
            st.store(nk, nk + TL::ELEMS);
        }
        __syncthreads();
        cur ^= 1;
    }
    l = half_sum(l);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (!exists) return;
    const int64_t at = ((int64_t)b * a.Lq + qi) * a.H + head, stat = ((int64_t)b * a.H + head) * a.Lq + qi;
    float lse, lse_lo;
    two_sum(m_use, __builtin_amdgcn_logf(l), lse, lse_lo);      // log2
    if (a.splits > 1) {
        const int64_t per = (int64_t)a.B * a.Lq * a.H;
        store_owned<float, TL::DBLOCKS>(a.part_o + (split * per + at) * a.D, o, inv, a.D, h);
        if (h == 0) {
            a.part_lse[split * per + stat] = l == 0.0f ? -INFINITY : lse;
            a.part_lse[(a.splits + split) * per + stat] = l == 0.0f ? 0.0f : lse_lo;
        }
    } else {
        store_owned<T, TL::DBLOCKS>(static_cast<T*>(a.out) + at * a.D, o, inv, a.D, h);
        if constexpr (TWO_TERMS) store_owned<float, TL::DBLOCKS>(a.out_f32 + at * a.D, o, inv, a.D, h);
        if (TRAIN && h == 0) {
            a.lse[stat] = l == 0.0f ? INFINITY : lse;
            a.lse[(int64_t)a.B * a.Lq * a.H + stat] = l == 0.0f ? 0.0f : lse_lo;
        }
    }
}

// LDS of fwd_few_kernel before its bias columns: the waves' value tiles, later their sums
template <typename T, int DP>
__host__ __device__ constexpr size_t few_bytes(int rows) {
    const size_t tiles = 4 * sizeof(typename Parts<T>::Lds) * Tile<T, DP, 32>::ELEMS, sums = sizeof(float) * 4 * (2 * 32 + (size_t)rows * DP);
    return tiles > sums ? tiles : sums;
}

// Few queries without a gradient (at most 32 rows with those of the heads that share keys: single tokens).  The rows fill one wave, and in
// fwd_kernel the other three would only fetch for it.  Here every wave holds the same rows and takes every fourth tile of 32 keys by itself:
// keys go from memory straight into the A operand, values through a wave's own piece of LDS (for the transposing read), no barrier until
// the waves' sums are joined.  Bound by reading keys and values: 16 single tokens of 8 heads of 64 over 0 .. 16384 keys of 2 shared heads
// (67 MB, bf16) 21.3 us with the join, 3.1 TB/s (fwd_kernel: 24.9); two tiles in flight instead of one: 22.1, 1024 workgroups instead of 512: 23.5.
template <typename T, int DP, int AXES>
__global__ __launch_bounds__(256, DP == 128 ? 1 : 2) void fwd_few_kernel(Args a) {
    using TL = Tile<T, DP, 32>;
    using L = typename TL::Lds;
    constexpr int WAVES = 4, THREADS = 64 * WAVES, ENTRY = (int)sizeof(float), N = 32 * TL::CHUNKS / 64, C = TL::E * sizeof(T) / 16;
    extern __shared__ __align__(16) char smem[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    const int groups = a.H / a.pack;
    const int split = blockIdx.x % a.splits, id = blockIdx.x / a.splits;       // pieces of a sample share nothing: spread over the XCDs
    const int hh = id % groups, b = id / groups, kvh = hh * a.pack / (a.H / a.Hk);
    const int rows = a.pack * a.Lq, row = lane & 31;
    const bool exists = row < rows;
    const int sub = exists ? row / a.Lq : 0, qi = exists ? row - sub * a.Lq : 0, head = hh * a.pack + sub;
    L* vt = reinterpret_cast<L*>(smem) + wave * TL::ELEMS;
    float* lut = reinterpret_cast<float*>(smem + few_bytes<T, DP>(rows));

    const int len = kept_length(a, b), n_tiles = (len + 31) / 32;
    const int t0 = split * a.tiles_per_split, t1 = min(n_tiles, t0 + a.tiles_per_split);
    const T* kp = static_cast<const T*>(a.k) + b * a.ks.b + kvh * a.ks.h;
    const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + kvh * a.vs.h;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_bs : nullptr;

    Frag<T> qf[TL::KSTEPS];
    load_owned<T, DP>(qf, static_cast<const T*>(a.q) + b * a.qs.b + qi * a.qs.l + head * a.qs.h, exists, a.D, h);
    int qa[AXES ? AXES : 1], lo[AXES ? AXES : 1], hi[AXES ? AXES : 1];
    const int* kpos = nullptr;
    if constexpr (AXES > 0) {
        fill_lut<AXES, THREADS>(a.rb, lut, hh * a.pack, a.pack, a.H);
        __syncthreads();
        kpos = a.rb.kpos + b * a.rb.kpos_bs;
#pragma unroll
        for (int x = 0; x < AXES; ++x) {
            const int centre = (int)lds_address(lut + (sub * AXES + x) * (2 * a.rb.limit + 1) + a.rb.limit);
            qa[x] = centre + scale_pos<-ENTRY>(a.rb.qpos[b * a.rb.qpos_bs + (int64_t)qi * AXES + x]);
            lo[x] = centre - ENTRY * a.rb.limit;
            hi[x] = centre + ENTRY * a.rb.limit;
        }
    }
    const LaneMap<TL, T> map(lane);

    // on its way from memory: the lane's row of keys (of the last key where there is none: masked below), its chunks of values
    struct InFlight {
        chunk16 k[TL::KSTEPS][C], v[N][C];
        StreamPos<AXES, 1, ENTRY> pos;
    };
    auto load = [&](InFlight& in, int t) {
        const T* k = kp + (int64_t)min(t * 32 + row, len - 1) * a.ks.l;
#pragma unroll
        for (int s = 0; s < TL::KSTEPS; ++s) {
            const int c = (2 * s + h) * TL::E;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                in.k[s][i] = chunk16{0, 0, 0, 0};
                if (c < a.D) in.k[s][i] = reinterpret_cast<const chunk16*>(k + c)[i];
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int f = lane + 64 * n, c = f % TL::CHUNKS * TL::E;
            const T* v = vp + (int64_t)min(t * 32 + f / TL::CHUNKS, len - 1) * a.vs.l + c;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                in.v[n][i] = chunk16{0, 0, 0, 0};
                if (c < a.D) in.v[n][i] = reinterpret_cast<const chunk16*>(v)[i];
            }
        }
        if constexpr (AXES > 0) in.pos.load(kpos, t * 32, len);
    };

    acc16 o[TL::DBLOCKS];
#pragma unroll
    for (int d = 0; d < TL::DBLOCKS; ++d) o[d] = acc16{0};
    float m = -INFINITY, m_use = 0.0f, l = 0.0f;
    InFlight in;
    if (t0 + wave < t1) load(in, t0 + wave);
    for (int t = t0 + wave; t < t1; t += WAVES) {
        const unsigned bits = (unsigned)kept_bits(mask, t * 32, len, 32);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int f = lane + 64 * n;
            put_chunk<T, TL>(vt + TL::chunk_at(f / TL::CHUNKS, f % TL::CHUNKS), in.v[n], (bits >> (f / TL::CHUNKS)) & 1);
        }
        acc16 s = acc16{0};
#pragma unroll
        for (int ks = 0; ks < TL::KSTEPS; ++ks) s = mma<T>(chunk_frag<T>(in.k[ks]), qf[ks], s);
        const StreamPos<AXES, 1, ENTRY> pos = in.pos;
        if (t + WAVES < t1) load(in, t + WAVES);
        if constexpr (AXES > 0) {
            int off[AXES][16];
#pragma unroll
            for (int x = 0; x < AXES; ++x) broadcast_plus(pos.p[0][x], qa[x], off[x]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = __builtin_fmaf(s[i], a.scale_log2, pair_bias<AXES>(off, i, lo, hi));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] *= a.scale_log2;
        }
        if (bits != 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = kept_row(bits, i) ? s[i] : -INFINITY;
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i]);
        if (__any(m == -INFINITY || top - m_use > exponent_limit<T>())) {
            top = half_max(top);
            const float mn = m == -INFINITY || top - m_use > exponent_limit<T>() ? fmaxf(m, top) : m;
            m_use = mn == -INFINITY ? 0.0f : mn;
            const float alpha = __builtin_amdgcn_exp2f(m - m_use);
#pragma unroll
            for (int d = 0; d < TL::DBLOCKS; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= alpha;
            l *= alpha;
            m = mn;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[i] = __builtin_amdgcn_exp2f(s[i] - m_use);
            l += s[i];
        }
        wave_order();       // the values are there for the other lanes
#pragma unroll
        for (int ps = 0; ps < TL::PSTEPS; ++ps) {
            const Frag<T> p = pack_step<T>(s, ps);
#pragma unroll
            for (int d = 0; d < TL::DBLOCKS; ++d) o[d] = mma<T>(map.read_col(vt, ps, d), p, o[d]);
        }
        wave_order();       // before the next tile's values take their place
    }
    l = half_sum(l);
    __syncthreads();
    // join the waves: [wave][rows][m, l], [wave][rows][DP]
    float* stat = reinterpret_cast<float*>(smem);
    float* sum = stat + WAVES * 2 * 32;
    if (exists) {
        if (h == 0) {
            stat[(wave * 32 + row) * 2] = m;
            stat[(wave * 32 + row) * 2 + 1] = l;
        }
        store_owned<float, TL::DBLOCKS>(sum + (wave * rows + row) * DP, o, 1.0f, a.D, h);
    }
    __syncthreads();
    const int64_t per = (int64_t)a.B * a.Lq * a.H;
    for (int f = tid; f < rows * (DP / 4); f += THREADS) {
        const int r = f / (DP / 4), c = f % (DP / 4) * 4;
        if (c >= a.D) continue;
        float M = -INFINITY, total = 0.0f, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) M = fmaxf(M, stat[(w * 32 + r) * 2]);
        const float use = M == -INFINITY ? 0.0f : M;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float g = __builtin_amdgcn_exp2f(stat[(w * 32 + r) * 2] - use);
            total = __builtin_fmaf(g, stat[(w * 32 + r) * 2 + 1], total);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(g, sum[(w * rows + r) * DP + c + i], acc[i]);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= inv;
        const int rs = r / a.Lq, ri = r - rs * a.Lq, rh = hh * a.pack + rs;
        const int64_t at = ((int64_t)b * a.Lq + ri) * a.H + rh;
        if (a.splits > 1) {
            store_f32<float, 4>(a.part_o + (split * per + at) * a.D + c, acc);
            if (c == 0) {
                float lse, lse_lo;
                two_sum(use, __builtin_amdgcn_logf(total), lse, lse_lo);
                float* part = a.part_lse + split * per + ((int64_t)b * a.H + rh) * a.Lq + ri;
                part[0] = total == 0.0f ? -INFINITY : lse;
                part[a.splits * per] = total == 0.0f ? 0.0f : lse_lo;
            }
        } else {
            store_f32<T, 4>(static_cast<T*>(a.out) + at * a.D + c, acc);
        }
    }
}

// Joins the splits of the forward.  A wave per row: `lanes` (a power of two >= D / 4) lanes hold 4 elements each, the 64 / lanes groups
// take every (64 / lanes)-th split, and the groups are added at the end -- with one group, 64 splits would be 64 dependent loads.
// (128 rows of 64, 16 parts: 4.4 us, latency; 16384 rows of 32, 4 parts in fp32: 10.5 us.)
template <typename T>
__global__ __launch_bounds__(256) void fwd_join_kernel(Args a, int lanes) {
    const int64_t rows = (int64_t)a.B * a.Lq * a.H, at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= rows) return;
    const int lane = threadIdx.x & 63, c = (lane & (lanes - 1)) * 4, group = lane / lanes, groups = 64 / lanes;
    const int head = (int)(at % a.H);
    const int64_t bq = at / a.H;
    const int64_t stat = ((bq / a.Lq) * a.H + head) * a.Lq + bq % a.Lq;
    const float *part = a.part_lse + stat, *part_lo = part + a.splits * rows;
    float top = -INFINITY, use_lo = 0.0f;
    bool bad = false;
    for (int s = lane; s < a.splits; s += 64) {
        const float v = part[s * rows];
        top = fmaxf(top, v);
        bad |= v != v;
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const bool far = is_far(top);
    if (far) {          // the second term of the highest, so that no weight passes 1
        use_lo = -INFINITY;
        for (int s = lane; s < a.splits; s += 64)
            if (part[s * rows] == top) use_lo = fmaxf(use_lo, part_lo[s * rows]);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) use_lo = fmaxf(use_lo, __shfl_xor(use_lo, off, 64));
    }
    bad = __any(bad);
    const float use = top == -INFINITY ? 0.0f : top;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sum = 0.0f;
    auto add_up = [&](auto far_rows) {
#pragma unroll 4
        for (int s = group; s < a.splits; s += groups) {
            float w = part[s * rows] - use, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (decltype(far_rows)::value) w += part_lo[s * rows] - use_lo;
            w = __builtin_amdgcn_exp2f(w);
            if (c < a.D && w != 0.0f) load_f32<float, 4>(a.part_o + (s * rows + at) * a.D + c, v);
            sum += w;
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(w, v[i], acc[i]);
        }
    };
    if (far) add_up(Int<1>{});
    else add_up(Int<0>{});
    for (int off = 32; off >= lanes; off >>= 1) {
        sum += __shfl_xor(sum, off, 64);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += __shfl_xor(acc[i], off, 64);
    }
    if (group != 0) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (a.lse && c == 0) {
        float lse, lse_lo;
        two_sum(use, use_lo + __builtin_amdgcn_logf(sum), lse, lse_lo);
        a.lse[stat] = bad ? NAN : sum == 0.0f ? INFINITY : lse;
        a.lse[rows + stat] = sum == 0.0f ? 0.0f : lse_lo;
    }
    if (c >= a.D) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = bad ? NAN : acc[i] * inv;
    store_f32<T, 4>(static_cast<T*>(a.out) + at * a.D + c, acc);
    if (a.out_f32) store_f32<float, 4>(a.out_f32 + at * a.D + c, acc);
}

// power of two that brings x to 2^14 .. 2^15 (1 for zero, infinity and NaN)
__device__ __forceinline__ float bound_scale(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 255) - 127;
    return x > 0.0f && e < 128 ? __uint_as_float((unsigned)(min(127 + 14 - e, 254)) << 23) : 1.0f;
}

// largest |v| of a kv head's kept keys, for whole waves
__device__ __forceinline__ float values_max(const Args& a, int b, int kvh) {
    const int lane = threadIdx.x & 63;
    float x = lane < a.v_chunks ? a.v_max[((int64_t)b * a.Hk + kvh) * a.v_chunks + lane] : 0.0f;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
    return x;
}

// v_max: a workgroup per chunk of a kv head's keys, of 128 or a 64th of them.  (3 x 1237 keys of 2 heads of 40: 4.7 us, a launch.)
constexpr int MAX_V_CHUNKS = 64;
inline int v_chunks(const Args& a) {
    const int n = (a.Lk + 127) / 128;
    return n < MAX_V_CHUNKS ? n : MAX_V_CHUNKS;
}
template <typename T>
__global__ __launch_bounds__(256) void values_max_kernel(Args a) {
    const int chunk = blockIdx.x % a.v_chunks, unit = blockIdx.x / a.v_chunks, kvh = unit % a.Hk, b = unit / a.Hk, len = kept_length(a, b);
    const int per = (a.Lk + a.v_chunks - 1) / a.v_chunks, row0 = chunk * per, rows = min(len - row0, per), vecs = a.D / 8;
    const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + kvh * a.vs.h;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_bs : nullptr;
    float x = 0.0f;
    const int step = 256 / vecs, c = (int)threadIdx.x % vecs * 8;       // threads beyond step * vecs have no part
#pragma unroll 4
    for (int r = (int)threadIdx.x / vecs; r < rows; r += step) {
        float v[8];
        load8(vp + (row0 + r) * a.vs.l + c, v);
        const bool kept = (int)threadIdx.x < step * vecs && (mask == nullptr || mask[row0 + r] != 0);
#pragma unroll
        for (int e = 0; e < 8; ++e) x = kept ? fmaxf(x, fabsf(v[e])) : x;
    }
    __shared__ float most[4];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
    if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = x;
    __syncthreads();
    if (threadIdx.x == 0) a.v_max[blockIdx.x] = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
}

// power of two that brings x to 1 .. 2 (1 for zero, infinity and NaN)
__device__ __forceinline__ float unit_scale(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 255) - 127;
    return x > 0.0f && e < 128 ? __uint_as_float((unsigned)(127 - e) << 23) : 1.0f;
}

// ------------------------------------------------------------------------------------------------------------ dq
constexpr int dkdv_stats(bool far_rows) { return far_rows ? 3 : 2; }       // numbers of a streamed row beside its tiles

// FAR_ROWS: scores are rounded as in the forward before both terms of lse are taken off them.  That is one or two instructions more a pair, and
// in a branch it displaces what the narrow kernels' registers are spent on (484 -> 506 to 576 us at the size below, taken or not; in dkdv 361
// -> 370, and 658 -> 780 for a whole step of fp32 heads of 64).  So both adjoints of far rows are a launch of their own (far_kernel): its
// workgroups leave at once (5 us), but for those of dq with a far row and those of dkdv whose kv head has one, which compute all their rows again.
// HIST: with the table's gradient.  LDS: tiles (one buffer), lut, hist[axes * buckets][columns].  A thread adds to a column by plain reads and
// writes: sums in a fixed order, no bank conflicts.  One axis: a column per thread, and 2 waves instead of 4 (WAVES) where more than 64
// buckets would not fit.  Two axes: lanes l and l + 32 share a column; they take the axes in opposite order, so that one is among the rows of
// the first axis while the other is among those of the second.  With that, 32-row tiles and eight registers' cells at a time three
// workgroups share a CU in narrow 16-bit heads, one computing while another waits at a barrier or for LDS.
// Measured with a two-axis bias of 2 x 32 buckets, 4 heads of 32: 8 x 8160 queries x 2048 keys, bf16: 480 us (a column per thread, two
// workgroups: 547; adding a block's ds while the next one is computed took 16 % of the vector instructions away and no time).  LDS and vector
// arithmetic are both busy 61 % of the time: waves wait for LDS reads and at barriers 45 % of their cycles, and the registers allow only three
// a SIMD to cover that.  2 x 2048 x 8160, fp32: 265 us (tiles in two buffers, one workgroup: 465 with fp32 products).
constexpr int hist_columns(int axes, int waves) { return axes == 2 ? 32 * waves : 64 * waves; }

// blocks: of the launch's workgroups those that work on this
template <typename T, int DP, int AXES, int WAVES, bool HIST, bool FAR_ROWS>
__device__ __forceinline__ void dq_body(const Args& a, int block, int blocks) {
    constexpr int R = dq_tile_rows(sizeof(T), DP, HIST);
    using TL = Tile<T, DP, R>;
    using L = typename TL::Lds;
    using Entry = __type_pack_element<HIST ? 1 : 0, float, Entry8>;
    constexpr int THREADS = 64 * WAVES, OWN = 32 * WAVES, ENTRY = (int)sizeof(Entry), COLS = hist_columns(AXES, WAVES);
    constexpr bool SHARED = HIST && AXES == 2;
    extern __shared__ __align__(16) char smem[];
    L* tiles = reinterpret_cast<L*>(smem);
    Entry* lut = reinterpret_cast<Entry*>(tiles + (HIST ? 2 : 4) * TL::ELEMS);
    const int span = 2 * a.rb.limit + 1, hist_rows = AXES * a.rb.buckets;
    float* hist = reinterpret_cast<float*>(lut + AXES * span);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int id = unit_per_xcd(block, blocks, a.row_tiles * a.splits);
    const int split = id % a.splits;
    id /= a.splits;
    const int rt = id % a.row_tiles;
    id /= a.row_tiles;
    const int head = id % a.H, b = id / a.H, kvh = head / (a.H / a.Hk);
    const int qi = rt * OWN + wave * 32 + (lane & 31);
    const bool exists = qi < a.Lq;
    const int q0 = exists ? qi : 0;
    const int half = SHARED ? h : 0;            // a lane's axis in turn x is x ^ half

    const int len = kept_length(a, b);
    const int n_tiles = (len + TL::ROWS - 1) / TL::ROWS;
    const int t0 = split * a.tiles_per_split;
    const int t1 = a.dq || HIST ? min(n_tiles, t0 + a.tiles_per_split) : t0;      // else only delta is wanted
    const T* kp = static_cast<const T*>(a.k) + b * a.ks.b + kvh * a.ks.h;
    const T* vp = static_cast<const T*>(a.v) + b * a.vs.b + kvh * a.vs.h;
    const unsigned char* mask = a.mask ? a.mask + b * a.mask_bs : nullptr;
    const int64_t at = ((int64_t)b * a.Lq + q0) * a.H + head, stat = ((int64_t)b * a.H + head) * a.Lq + q0;

    Frag<T> qf[TL::KSTEPS], gf[TL::KSTEPS];
    load_owned<T, DP>(qf, static_cast<const T*>(a.q) + b * a.qs.b + q0 * a.qs.l + head * a.qs.h, exists, a.D, h);
    const float sign = dp_sign<T>(lane);
    load_owned<T, DP>(gf, static_cast<const T*>(a.go) + at * a.D, exists, a.D, h, sign);
    float delta = 0.0f, most = 0.0f, l1 = 0.0f;
#pragma unroll
    for (int ks = 0; ks < TL::KSTEPS; ++ks) {
        const int c = (2 * ks + h) * TL::E;
        if (exists && c < a.D) {
            float g[8], o[8];
            load8(static_cast<const T*>(a.go) + at * a.D + c, g);
            load8(a.o + at * a.D + c, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(o[e], g[e], delta);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                most = fmaxf(most, fabsf(g[e]));
                l1 += fabsf(g[e]);
            }
        }
    }
    delta = half_sum(delta);
    if (!FAR_ROWS && exists && split == 0 && h == 0) a.delta[stat] = delta;
    float unscale = 1.0f, p_log2 = 0.0f;       // p is taken times 2^p_log2
    if constexpr (__is_same(T, _Float16)) {
        most = half_max(most);
        l1 = half_sum(l1);
        if (!FAR_ROWS && exists && split == 0 && h == 0) a.go_l1[stat] = l1;
        const float f = unit_scale(most), fp = bound_scale(2.0f * l1 * f * values_max(a, b, kvh));
        unscale = unit_scale(f) * unit_scale(fp);
        p_log2 = (float)(((int)__float_as_uint(fp) >> 23) - 127);
        delta *= f;
#pragma unroll
        for (int s = 0; s < TL::KSTEPS; ++s)
#pragma unroll
            for (int e = 0; e < TL::E; ++e) gf[s].part[0][e] = (T)((float)gf[s].part[0][e] * f);
    }
    // the accumulators start at -lse / scale and -delta: the products come out as the exponent and as dp - D.  +inf (a row without keys,
    // or none at all) makes every p zero.
    constexpr bool FOLD = fold_start<T>(), FOLD_S = FOLD && !FAR_ROWS;
    const float lse = exists ? a.lse[stat] : INFINITY;
    const float lse_lo = (FAR_ROWS ? a.lse[(int64_t)a.B * a.H * a.Lq + stat] : 0.0f) - p_log2;
    if constexpr (!FAR_ROWS) {
        const bool far = __any(is_far(lse));
        if (split == 0 && lane == 0) a.far_rows[((int64_t)b * a.H + head) * a.row_groups + rt * WAVES + wave] = far;
    }
    const acc16 start_s = FOLD_S ? splat((p_log2 - lse) / a.scale_log2) : acc16{0}, start_d = FOLD ? splat(-delta) : acc16{0};
    const LaneMap<TL, T> map(lane);
    int qa[AXES ? AXES : 1], lo[AXES ? AXES : 1], hi[AXES ? AXES : 1];
    const int* kpos = nullptr;
    if constexpr (AXES > 0) {
        fill_lut<AXES, THREADS>(a.rb, lut, head, HIST ? 4 * COLS : 1, a.H);
        kpos = a.rb.kpos + b * a.rb.kpos_bs;
#pragma unroll
        for (int x = 0; x < AXES; ++x) {
            const int centre = (int)lds_address(lut + (x ^ half) * span + a.rb.limit);
            qa[x] = centre + scale_pos<-ENTRY>(a.rb.qpos[b * a.rb.qpos_bs + (int64_t)q0 * AXES + (x ^ half)]);
            lo[x] = centre - ENTRY * a.rb.limit;
            hi[x] = centre + ENTRY * a.rb.limit;
        }
        if constexpr (HIST)
            for (int i = tid; i < hist_rows * COLS; i += THREADS) hist[i] = 0.0f;
    }
    char* column = reinterpret_cast<char*>(hist + (SHARED ? wave * 32 + (lane & 31) : tid));

    acc16 dq[TL::DBLOCKS];
#pragma unroll
    for (int d = 0; d < TL::DBLOCKS; ++d) dq[d] = acc16{0};
    Stream<T, DP, R, THREADS> st;
    StreamPos<AXES, TL::BLOCKS, ENTRY> pos, pos_next;
    st.init(a.ks.l, a.vs.l);
    int cur = 0;
    if (t0 < t1) {
        st.load(kp + t0 * (int64_t)TL::ROWS * a.ks.l, vp + t0 * (int64_t)TL::ROWS * a.vs.l, t0 * TL::ROWS, len, a.D, mask);
        if constexpr (AXES > 0) pos_next.template load<SHARED>(kpos, t0 * TL::ROWS, len);
        st.store(tiles, tiles + TL::ELEMS);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const unsigned long long bits = kept_bits(mask, t * TL::ROWS, len, TL::ROWS);
        if constexpr (AXES > 0) pos = pos_next;
        if (t + 1 < t1) {
            st.load(kp + (t + 1) * (int64_t)TL::ROWS * a.ks.l, vp + (t + 1) * (int64_t)TL::ROWS * a.vs.l, (t + 1) * TL::ROWS, len, a.D, mask);
            if constexpr (AXES > 0) pos_next.template load<SHARED>(kpos, (t + 1) * TL::ROWS, len);
        }
        const L *kt = HIST ? tiles : tiles + cur * 2 * TL::ELEMS, *vt = kt + TL::ELEMS;
#pragma unroll
        for (int nb = 0; nb < TL::BLOCKS; ++nb) {
            const unsigned half_bits = (unsigned)(bits >> (nb * 32));
            if (half_bits == 0) continue;
            const L *kb = kt + nb * 32 * DP, *vb = vt + nb * 32 * DP;
            acc16 s = product<T, TL>(map, kb, qf, start_s), dp = product<T, TL>(map, vb, gf, start_d);
            if constexpr (HIST) {
                auto octet = [&](auto which) {      // eight registers at a time: their cells' places need not all be held at once
                    constexpr int F = decltype(which)::value;
                    int off[AXES][8];
                    unsigned at[8][AXES];
#pragma unroll
                    for (int x = 0; x < AXES; ++x) broadcast_plus8<F>(pos.p[nb][x], qa[x], off[x]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int i = F + k;
                        float bias = 0.0f;
#pragma unroll
                        for (int x = 0; x < AXES; ++x) {
                            const uint2v e = lds_load<uint2v>(med3(off[x][k], lo[x], hi[x]));       // an Entry8
                            bias = x ? bias + __uint_as_float(e[0]) : __uint_as_float(e[0]);
                            at[k][x] = e[1];
                        }
                        s[i] = __builtin_fmaf(s[i], a.scale_log2, bias);
                        if constexpr (!FOLD_S) s[i] -= lse;
                        if constexpr (FAR_ROWS) s[i] -= lse_lo;
                        s[i] = kept_row(half_bits, i) ? s[i] : -INFINITY;
                        dp[i] = (FOLD ? dp[i] : __builtin_fmaf(dp[i], sign, -delta)) * __builtin_amdgcn_exp2f(s[i]);
                    }
#pragma unroll
                    for (int x = 0; x < AXES; ++x) {
#pragma unroll
                        for (int k = 0; k < 8; k += 2) {
                            const float d0 = __is_same(T, _Float16) ? dp[F + k] * unscale : dp[F + k], d1 = __is_same(T, _Float16) ? dp[F + k + 1] * unscale : dp[F + k + 1];
                            hist_add2(column, at[k][x], d0, at[k + 1][x], d1);
                        }
                        if constexpr (SHARED) wave_order();         // the halves change axes
                    }
                };
                octet(Int<0>{});
                octet(Int<8>{});
            } else {
                int off[AXES ? AXES : 1][16];
#pragma unroll
                for (int x = 0; x < AXES; ++x) broadcast_plus(pos.p[nb][x], qa[x], off[x]);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if constexpr (AXES > 0) {
                        s[i] = __builtin_fmaf(s[i], a.scale_log2, pair_bias<AXES>(off, i, lo, hi));
                        if constexpr (!FOLD_S) s[i] -= lse;
                    } else if constexpr (FAR_ROWS) {
                        s[i] = s[i] * a.scale_log2 - lse;
                    } else {
                        s[i] = FOLD ? s[i] * a.scale_log2 : __builtin_fmaf(s[i], a.scale_log2, -lse);
                    }
                    if constexpr (FAR_ROWS) s[i] -= lse_lo;
                }
                if (half_bits != 0xffffffffu) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = kept_row(half_bits, i) ? s[i] : -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] = (FOLD ? dp[i] : __builtin_fmaf(dp[i], sign, -delta)) * __builtin_amdgcn_exp2f(s[i]);
            }
#pragma unroll
            for (int ps = 0; ps < TL::PSTEPS; ++ps) {
                const Frag<T> p = pack_step<T>(dp, ps);
#pragma unroll
                for (int d = 0; d < TL::DBLOCKS; ++d) dq[d] = mma<T>(map.read_col(kb, ps, d), p, dq[d]);
            }
        }
        if constexpr (HIST) __syncthreads();
        if (t + 1 < t1) {
            L* nk = HIST ? tiles : tiles + (cur ^ 1) * 2 * TL::ELEMS;
            st.store(nk, nk + TL::ELEMS);
        }
        __syncthreads();
        cur ^= 1;
    }
    if (a.dq && exists) {
        if (a.splits > 1) store_owned<float, TL::DBLOCKS>(a.part_o + ((int64_t)split * a.B * a.Lq * a.H + at) * a.D, dq, a.scale * unscale, a.D, h);
        else store_owned<T, TL::DBLOCKS>(static_cast<T*>(a.dq) + at * a.D, dq, a.scale * unscale, a.D, h);
    }
    if constexpr (HIST) {       // rows that do not exist added zeros
        const int64_t part = ((int64_t)b * a.row_tiles + rt) * a.splits + split;
        for (int n = wave; n < hist_rows; n += WAVES) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < COLS / 64; ++k) v += hist[n * COLS + k * 64 + lane];
            v = wave_sum(v);
            if (lane == 0) a.part_table[((int64_t)head * a.parts + part) * hist_rows + n] = v;
        }
    }
}

template <typename T, int DP, int AXES, int WAVES, bool HIST>
__global__ __launch_bounds__(64 * WAVES, DP == 32 ? ((!HIST && AXES == 2) || sizeof(T) == 4 ? 2 : 3) : DP == 64 && !(HIST && sizeof(T) == 4) ? 2 : 1) void dq_kernel(Args a) { dq_body<T, DP, AXES, WAVES, HIST, false>(a, blockIdx.x, gridDim.x); }

// ------------------------------------------------------------------------------------------------------------ dk, dv
// Measured at the sizes above: bf16 360 us (LDS busy 57 % of the time, vector arithmetic 52 %; waves wait 43 % of their cycles for LDS reads and at
// barriers, three of them on a SIMD), fp32 250 us.
template <typename T, int DP, int AXES, bool FAR_ROWS>
__device__ __forceinline__ void dkdv_body(const Args& a, int block, int blocks) {
    constexpr int R = tile_rows(sizeof(T), DP);
    using TL = Tile<T, DP, R>;
    using L = typename TL::Lds;
    constexpr int THREADS = 256, ENTRY = (int)sizeof(float), STATS = dkdv_stats(FAR_ROWS);
    extern __shared__ __align__(16) char smem[];
    L* tiles = reinterpret_cast<L*>(smem);                                              // [2][Q, dO]
    float* stats = reinterpret_cast<float*>(tiles + 4 * TL::ELEMS);                     // [2][lse, delta (FAR_ROWS: and lse's second term)][ROWS]
    float* lut = reinterpret_cast<float*>(stats + 2 * STATS * TL::ROWS);

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5;
    int id = unit_per_xcd(block, blocks, a.row_tiles * a.splits);
    const int split = id % a.splits;
    id /= a.splits;
    const int rt = id % a.row_tiles;
    id /= a.row_tiles;
    const int kvh = id % a.Hk, b = id / a.Hk, group = a.H / a.Hk;
    const int kj = rt * 128 + wave * 32 + (lane & 31);
    const int len = kept_length(a, b);
    bool kept = kj < len;
    if (kept && a.mask) kept = a.mask[b * a.mask_bs + kj] != 0;
    const LaneMap<TL, T> map(lane);

    Frag<T> kf[TL::KSTEPS], vf[TL::KSTEPS];
    const float sign = dp_sign<T>(lane);
    load_owned<T, DP>(kf, static_cast<const T*>(a.k) + b * a.ks.b + (int64_t)kj * a.ks.l + kvh * a.ks.h, kept, a.D, h);
    load_owned<T, DP>(vf, static_cast<const T*>(a.v) + b * a.vs.b + (int64_t)kj * a.vs.l + kvh * a.vs.h, kept, a.D, h, sign);
    int ka[AXES ? AXES : 1], lo[AXES ? AXES : 1], hi[AXES ? AXES : 1];
    const int* qpos = nullptr;
    if constexpr (AXES > 0) {
        qpos = a.rb.qpos + b * a.rb.qpos_bs;
#pragma unroll
        for (int x = 0; x < AXES; ++x) {
            const int centre = (int)lds_address(lut + x * (2 * a.rb.limit + 1) + a.rb.limit);
            ka[x] = (kept ? scale_pos<ENTRY>(a.rb.kpos[b * a.rb.kpos_bs + (int64_t)kj * AXES + x]) : 0) + centre;
            lo[x] = centre - ENTRY * a.rb.limit;
            hi[x] = centre + ENTRY * a.rb.limit;
        }
    }
    constexpr bool HALF = __is_same(T, _Float16), FOLD = fold_start<T>(), FOLD_S = FOLD && !FAR_ROWS;
    constexpr float P_LOG2 = HALF ? 10.0f : 0.0f, P_UNSCALE = HALF ? 1.0f / 1024.0f : 1.0f;
    float ds_scale = 1.0f, ds_unscale = 1.0f;       // of dS beside that of P
    if constexpr (HALF) {
        __shared__ float most[THREADS / 64];
        float x = 0.0f;
        const float* rows = a.go_l1 + ((int64_t)b * a.H + kvh * group) * a.Lq;
        const int64_t n = (int64_t)group * a.Lq;
        for (int64_t i = tid; i < n; i += THREADS) x = fmaxf(x, rows[i]);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) x = fmaxf(x, __shfl_xor(x, off, 64));
        if (lane == 0) most[wave] = x;
        __syncthreads();
        const float f = bound_scale(2.0f * fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3])) * values_max(a, b, kvh));
        ds_scale = f * P_UNSCALE;
        ds_unscale = unit_scale(f);
    }
    acc16 dk[TL::DBLOCKS], dv[TL::DBLOCKS];
#pragma unroll
    for (int d = 0; d < TL::DBLOCKS; ++d) dk[d] = dv[d] = acc16{0};

    // the streamed sequence: query tiles of every head of the group, one after the other
    const int q_tiles = (a.Lq + TL::ROWS - 1) / TL::ROWS, n_tiles = q_tiles * group;
    const int t0 = split * a.tiles_per_split;
    int t1 = min(n_tiles, t0 + a.tiles_per_split);
    if (rt * 128 >= len) t1 = t0;        // no key of this workgroup is kept: zeros
    Stream<T, DP, R, THREADS> st;
    StreamPos<AXES, TL::BLOCKS, -ENTRY> pos, pos_next;
    st.init(a.qs.l, (int64_t)a.H * a.D);
    float snext = 0.0f;
    int cur = 0;
    auto load = [&](int t) {
        const int head = kvh * group + t / q_tiles, row0 = (t % q_tiles) * TL::ROWS;
        st.load(static_cast<const T*>(a.q) + b * a.qs.b + head * a.qs.h + row0 * a.qs.l,
                static_cast<const T*>(a.go) + (((int64_t)b * a.Lq + row0) * a.H + head) * a.D, row0, a.Lq, a.D, nullptr);
        if (tid < STATS * TL::ROWS) {
            const int r = row0 + tid % TL::ROWS, which = tid / TL::ROWS;
            const float* src = which == 1 ? a.delta : a.lse + (which == 2 ? (int64_t)a.B * a.H * a.Lq : 0);
            // what the accumulators start at: -lse / scale (fp32 and FAR_ROWS: -lse, added at the end) and -delta; a row that does not exist has
            // lse = +inf, so p = 0
            const float x = r < a.Lq ? src[((int64_t)b * a.H + head) * a.Lq + r] : which == 0 ? INFINITY : 0.0f;
            snext = which == 0 && FOLD_S ? (P_LOG2 - x) / a.scale_log2 : -x;
        }
        if constexpr (AXES > 0) pos_next.load(qpos, row0, a.Lq);
    };
    auto store = [&](int buf) {
        L* n = tiles + buf * 2 * TL::ELEMS;
        st.store(n, n + TL::ELEMS);
        if (tid < STATS * TL::ROWS) stats[buf * STATS * TL::ROWS + tid] = snext;
    };
    int lut_head = -1;
    if (t0 < t1) {
        load(t0);
        store(0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        if constexpr (AXES > 0) pos = pos_next;
        if (t + 1 < t1) load(t + 1);
        if constexpr (AXES > 0) {
            const int head = kvh * group + t / q_tiles;
            if (head != lut_head) {     // the barrier at the end of the last round has ended every read of the old columns
                fill_lut<AXES, THREADS>(a.rb, lut, head, 1, a.H);
                lut_head = head;
                __syncthreads();
            }
        }
        const L *qt = tiles + cur * 2 * TL::ELEMS, *gt = qt + TL::ELEMS;
        const float* start = stats + cur * STATS * TL::ROWS;
#pragma unroll
        for (int nb = 0; nb < TL::BLOCKS; ++nb) {
            const L *qb = qt + nb * 32 * DP, *gb = gt + nb * 32 * DP;
            acc16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int r = nb * 32 + acc_row(i, h);
                s[i] = FOLD_S ? start[r] : 0.0f;
                dp[i] = FOLD ? start[TL::ROWS + r] : 0.0f;
            }
            s = product<T, TL>(map, qb, kf, s);
            dp = product<T, TL>(map, gb, vf, dp);
            int off[AXES ? AXES : 1][16];
#pragma unroll
            for (int x = 0; x < AXES; ++x) broadcast_plus(pos.p[nb][x], ka[x], off[x]);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float x;
                if constexpr (AXES > 0) {
                    x = __builtin_fmaf(s[i], a.scale_log2, pair_bias<AXES>(off, i, lo, hi));
                } else {
                    x = s[i] * a.scale_log2;
                }
                if constexpr (!FOLD_S) x += start[nb * 32 + acc_row(i, h)];
                if constexpr (FAR_ROWS) x += start[2 * TL::ROWS + nb * 32 + acc_row(i, h)] + P_LOG2;
                if constexpr (!FOLD) {
                    dp[i] = __builtin_fmaf(dp[i], sign, start[TL::ROWS + nb * 32 + acc_row(i, h)]);
                }
                s[i] = __builtin_amdgcn_exp2f(x);
                dp[i] *= HALF ? s[i] * ds_scale : s[i];
            }
#pragma unroll
            for (int ps = 0; ps < TL::PSTEPS; ++ps) {
                const Frag<T> p = pack_step<T>(s, ps), ds = pack_step<T>(dp, ps);
#pragma unroll
                for (int d = 0; d < TL::DBLOCKS; ++d) {
                    dv[d] = mma<T>(map.read_col(gb, ps, d), p, dv[d]);
                    dk[d] = mma<T>(map.read_col(qb, ps, d), ds, dk[d]);
                }
            }
        }
        if (t + 1 < t1) store(cur ^ 1);
        __syncthreads();
        cur ^= 1;
    }
    if (kj >= a.Lk) return;
    if (!kept) {        // a masked key's column of P was computed from zeros and is nobody else's
#pragma unroll
        for (int d = 0; d < TL::DBLOCKS; ++d) dk[d] = dv[d] = acc16{0};
    }
    const int64_t at = ((int64_t)b * a.Lk + kj) * a.Hk + kvh;
    if (a.splits > 1) {
        const int64_t off = (int64_t)split * a.B * a.Lk * a.Hk;
        store_owned<float, TL::DBLOCKS>(a.part_dk + (off + at) * a.D, dk, a.scale * ds_unscale, a.D, h);
        store_owned<float, TL::DBLOCKS>(a.part_dv + (off + at) * a.D, dv, P_UNSCALE, a.D, h);
    } else {
        store_owned<T, TL::DBLOCKS>(static_cast<T*>(a.dk) + at * a.D, dk, a.scale * ds_unscale, a.D, h);
        store_owned<T, TL::DBLOCKS>(static_cast<T*>(a.dv) + at * a.D, dv, P_UNSCALE, a.D, h);
    }
}

template <typename T, int DP, int AXES>
__global__ __launch_bounds__(256, DP == 32 ? (sizeof(T) == 2 ? 3 : 2) : DP == 64 ? 2 : 1) void dkdv_kernel(Args a) { dkdv_body<T, DP, AXES, false>(a, blockIdx.x, gridDim.x); }

// Both adjoints of far rows: dq's workgroups first.
template <typename T, int DP, int AXES, int WAVES, bool HIST>
__global__ __launch_bounds__(256, 1) void far_kernel(Args dq, Args dkdv, int dq_blocks) {
    // every wave looks for itself
    auto none = [](const int* rows, int n) {
        bool any = false;
        for (int i = threadIdx.x & 63; i < n; i += 64) any |= rows[i] != 0;
        return !__any(any);
    };
    int block = blockIdx.x;
    if (block < dq_blocks) {
        const int id = unit_per_xcd(block, dq_blocks, dq.row_tiles * dq.splits) / dq.splits;
        if (none(dq.far_rows + (int64_t)(id / dq.row_tiles) * dq.row_groups + id % dq.row_tiles * WAVES, WAVES)) return;
        dq_body<T, DP, AXES, WAVES, HIST, true>(dq, block, dq_blocks);
    } else {
        block -= dq_blocks;
        const int blocks = gridDim.x - dq_blocks, id = unit_per_xcd(block, blocks, dkdv.row_tiles * dkdv.splits) / dkdv.splits, n = dkdv.H / dkdv.Hk * dkdv.row_groups;
        if (none(dkdv.far_rows + (int64_t)(id / dkdv.row_tiles) * n, n)) return;
        dkdv_body<T, DP, AXES, true>(dkdv, block, blocks);
    }
}

// Everything the splits of the backward left to add, in one launch: out[n] = sum of a job's parts, in order, 4 elements a thread (n is a
// multiple of 8).  Jobs: dq, dk, dv; blockIdx.y selects.
struct SumJob {
    const float* part;
    void* out;
    int64_t n;
    int splits;
};
struct SumJobs {
    SumJob job[3];
};
template <typename T>
__global__ __launch_bounds__(256) void sum_parts_kernel(SumJobs jobs) {
    const SumJob j = jobs.job[blockIdx.y];
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= j.n) return;
    float acc[4], v[4];
    load_f32<float, 4>(j.part + i, acc);
#pragma unroll 4
    for (int s = 1; s < j.splits; ++s) {
        load_f32<float, 4>(j.part + s * j.n + i, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += v[e];
    }
    store_f32<T, 4>(static_cast<T*>(j.out) + i, acc);
}

// ------------------------------------------------------------------------------------------------------------ launches
constexpr size_t MAX_LDS = 159 * 1024;      // of a CU's 160 KB; the bias borders are static

template <typename T, int DP, int R>
constexpr size_t tile_bytes() { return 4 * sizeof(typename Parts<T>::Lds) * Tile<T, DP, R>::ELEMS; }

inline size_t lut_bytes(const Args& a, int axes, int heads) { return axes ? sizeof(float) * heads * axes * (2 * a.rb.limit + 1) : 0; }

template <typename K, typename... A>
int start(K kernel, const char* what, unsigned long long& done, dim3 grid, int threads, size_t lds, hipStream_t s, const A&... args) {
    if (lds > MAX_LDS || !camli_reserve_lds((const void*)kernel, MAX_LDS, done)) {
        camli_set_error("%s: cannot reserve %zu bytes of LDS", what, lds);
        return CAMLI_ELAUNCH;
    }
    kernel<<<grid, threads, lds, s>>>(args...);
    return camli_check_launch(what);
}

template <typename T, int DP, int AXES, bool TRAIN>
int run_fwd_mode(const Args& a, hipStream_t s) {
    constexpr int R = tile_rows(sizeof(T), DP);
    static unsigned long long done = 0;
    const size_t lds = tile_bytes<T, DP, R>() + lut_bytes(a, AXES, a.pack);
    return start(fwd_kernel<T, DP, AXES, TRAIN>, "camli_cross_attention_fwd", done, dim3(a.row_tiles * (a.H / a.pack) * a.B * a.splits), 256, lds, s, a);
}

template <typename T, int DP, int AXES>
int run_fwd_few(const Args& a, hipStream_t s) {
    static unsigned long long done = 0;
    const size_t lds = few_bytes<T, DP>(a.pack * a.Lq) + lut_bytes(a, AXES, a.pack);
    return start(fwd_few_kernel<T, DP, AXES>, "camli_cross_attention_fwd", done, dim3(a.H / a.pack * a.B * a.splits), 256, lds, s, a);
}

template <typename T, int DP, int AXES>
int run_fwd(const Args& a, hipStream_t s) {
    const int rc = a.few ? run_fwd_few<T, DP, AXES>(a, s) : a.lse ? run_fwd_mode<T, DP, AXES, true>(a, s) : run_fwd_mode<T, DP, AXES, false>(a, s);
    if (rc != CAMLI_OK || a.splits == 1) return rc;
    int lanes = 2;
    while (lanes * 4 < a.D) lanes *= 2;
    fwd_join_kernel<T><<<dim3((unsigned)(((int64_t)a.B * a.Lq * a.H + 3) / 4)), 256, 0, s>>>(a, lanes);
    return camli_check_launch("camli_cross_attention_fwd");
}

template <typename T, int DP, int AXES, int WAVES, bool HIST>
size_t dq_lds(const Args& a) {
    size_t lds = tile_bytes<T, DP, dq_tile_rows(sizeof(T), DP, HIST)>() / (HIST ? 2 : 1) + lut_bytes(a, AXES, 1);
    if (HIST) lds += lut_bytes(a, AXES, 1) + sizeof(float) * AXES * a.rb.buckets * hist_columns(AXES, WAVES);      // entries of 8 bytes
    return lds;
}
template <typename T, int DP, int AXES, bool FAR_ROWS>
size_t dkdv_lds(const Args& a) {
    constexpr int R = tile_rows(sizeof(T), DP);
    return tile_bytes<T, DP, R>() + sizeof(float) * 2 * dkdv_stats(FAR_ROWS) * R + lut_bytes(a, AXES, 1);
}

template <typename T, int DP, int AXES, int WAVES, bool HIST>
int run_dq_mode(const Args& a, hipStream_t s) {
    static unsigned long long done = 0;
    return start(dq_kernel<T, DP, AXES, WAVES, HIST>, "camli_cross_attention_bwd", done, dim3(a.row_tiles * a.H * a.B * a.splits), 64 * WAVES, dq_lds<T, DP, AXES, WAVES, HIST>(a), s, a);
}

template <typename T, int DP, int AXES, int WAVES, bool HIST>
int run_far_mode(const Args& dq, const Args& dkdv, hipStream_t s) {
    static unsigned long long done = 0;
    const int dq_blocks = dq.dq || HIST ? dq.row_tiles * dq.H * dq.B * dq.splits : 0, dkdv_blocks = dkdv.dk ? dkdv.row_tiles * dkdv.Hk * dkdv.B * dkdv.splits : 0;
    const size_t lq = dq_lds<T, DP, AXES, WAVES, HIST>(dq), lk = dkdv_lds<T, DP, AXES, true>(dkdv);
    auto launch = [&](int nq, int nk, int threads) {
        if (nq + nk == 0) return CAMLI_OK;
        return start(far_kernel<T, DP, AXES, WAVES, HIST>, "camli_cross_attention_bwd", done, dim3(nq + nk), threads, lq > lk ? lq : lk, s, dq, dkdv, nq);
    };
    if (WAVES == 4 && dq_blocks + dkdv_blocks < (1 << 24)) return launch(dq_blocks, dkdv_blocks, 256);      // 2^32 threads a launch
    const int rc = launch(dq_blocks, 0, 64 * WAVES);
    return rc == CAMLI_OK ? launch(0, dkdv_blocks, 256) : rc;
}

// RUN<..., WAVES, HIST> for what is wanted of the table's gradient
#define XATTN_SELECT_DQ(RUN, TABLE, ...)                                                                              \
    if constexpr (AXES > 0) {                                                                                         \
        if (!TABLE) return RUN<T, DP, AXES, 4, false>(__VA_ARGS__);                                                   \
        if constexpr (AXES == 1) return waves == 2 ? RUN<T, DP, AXES, 2, true>(__VA_ARGS__) : RUN<T, DP, AXES, 4, true>(__VA_ARGS__); \
        else return RUN<T, DP, AXES, 4, true>(__VA_ARGS__);                                                           \
    } else {                                                                                                          \
        return RUN<T, DP, AXES, 4, false>(__VA_ARGS__);                                                               \
    }

template <typename T, int DP, int AXES>
int run_dq(const Args& a, int waves, hipStream_t s) { XATTN_SELECT_DQ(run_dq_mode, a.part_table, a, s) }

template <typename T, int DP, int AXES>
int run_far(const Args& dq, const Args& dkdv, int waves, hipStream_t s) { XATTN_SELECT_DQ(run_far_mode, dq.part_table, dq, dkdv, s) }

template <typename T, int DP, int AXES>
int run_dkdv(const Args& a, hipStream_t s) {
    static unsigned long long done = 0;
    return start(dkdv_kernel<T, DP, AXES>, "camli_cross_attention_bwd", done, dim3(a.row_tiles * a.Hk * a.B * a.splits), 256, dkdv_lds<T, DP, AXES, false>(a), s, a);
}

// the kernels by head width (padded to 32, 64 or 128) and axes of the bias
template <typename T>
struct Launch {
    static int fwd(const Args& a, int axes, hipStream_t s);
    static int dq(const Args& a, int axes, int waves, hipStream_t s);
    static int dkdv(const Args& a, int axes, hipStream_t s);
    static int values(const Args& a, hipStream_t s);        // fp16 only
    static int far(const Args& dq, const Args& dkdv, int axes, int waves, hipStream_t s);
    static int sum(const SumJobs& jobs, int n, hipStream_t s);
};

#define XATTN_SELECT(RUN, ...)                                                                                      \
    if (a.D <= 32) return axes == 0 ? RUN<T, 32, 0>(__VA_ARGS__) : axes == 1 ? RUN<T, 32, 1>(__VA_ARGS__) : RUN<T, 32, 2>(__VA_ARGS__); \
    if (a.D <= 64) return axes == 0 ? RUN<T, 64, 0>(__VA_ARGS__) : axes == 1 ? RUN<T, 64, 1>(__VA_ARGS__) : RUN<T, 64, 2>(__VA_ARGS__); \
    return axes == 0 ? RUN<T, 128, 0>(__VA_ARGS__) : axes == 1 ? RUN<T, 128, 1>(__VA_ARGS__) : RUN<T, 128, 2>(__VA_ARGS__);

#define XATTN_DEFINE_FWD(TYPE) \
    template <> int Launch<TYPE>::fwd(const Args& a, int axes, hipStream_t s) { using T = TYPE; XATTN_SELECT(run_fwd, a, s) }
#define XATTN_DEFINE_DQ(TYPE) \
    template <> int Launch<TYPE>::dq(const Args& a, int axes, int waves, hipStream_t s) { using T = TYPE; XATTN_SELECT(run_dq, a, waves, s) }
#define XATTN_DEFINE_FAR(TYPE)                                                                                     \
    template <> int Launch<TYPE>::far(const Args& a, const Args& dkdv, int axes, int waves, hipStream_t s) {       \
        using T = TYPE;                                                                                            \
        XATTN_SELECT(run_far, a, dkdv, waves, s)                                                                   \
    }
#define XATTN_DEFINE_VALUES(TYPE)                                                                                  \
    template <> int Launch<TYPE>::values(const Args& a, hipStream_t s) {                                           \
        values_max_kernel<TYPE><<<dim3((unsigned)a.B * a.Hk * a.v_chunks), 256, 0, s>>>(a);                        \
        return camli_check_launch("camli_cross_attention_bwd");                                                    \
    }
#define XATTN_DEFINE_SUM(TYPE)                                                                                     \
    template <> int Launch<TYPE>::sum(const SumJobs& jobs, int n, hipStream_t s) {                                 \
        int64_t most = 0;                                                                                          \
        for (int i = 0; i < n; ++i) most = jobs.job[i].n > most ? jobs.job[i].n : most;                            \
        sum_parts_kernel<TYPE><<<dim3((unsigned)((most / 4 + 255) / 256), n), 256, 0, s>>>(jobs);                  \
        return camli_check_launch("camli_cross_attention_bwd");                                                    \
    }
#define XATTN_DEFINE_DKDV(TYPE) \
    template <> int Launch<TYPE>::dkdv(const Args& a, int axes, hipStream_t s) { using T = TYPE; XATTN_SELECT(run_dkdv, a, s) }

}  // namespace xattn
