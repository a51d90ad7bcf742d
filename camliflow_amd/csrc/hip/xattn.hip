// Cross attention: argument checks, work split and the C entries (kernels: xattn.h).
#include "xattn.h"

namespace {

using xattn::Args;

int padded(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }
int tile_rows(const Args& a, int type) { return xattn::tile_rows(camli_type_size(type), padded(a.D)); }

// Few owned rows leave CUs idle: the streamed side is cut until there are `want` workgroups, but into no less than `least_rows` rows a
// piece (a piece pays for its start and for its part of the join; fp32 rows take twice the time of 16-bit ones).
void split_stream(Args& a, int64_t base, int n_tiles, int tile, int want, int least_rows) {
    const int least = camli_divup(least_rows, tile);
    int splits = 1;
    if (base < want / 2) {
        splits = (int)((want + base - 1) / base);
        const int most = n_tiles / least < 1 ? 1 : n_tiles / least;
        if (splits > most) splits = most;
    }
    a.tiles_per_split = n_tiles ? (n_tiles + splits - 1) / splits : 1;
    a.splits = n_tiles ? (n_tiles + a.tiles_per_split - 1) / a.tiles_per_split : 1;
}

void plan_fwd(Args& a, int type, int axes, bool training) {
    const int group = a.H / a.Hk;
    // the query heads of a kv head share a workgroup where all their rows fit into one and their bias columns into LDS: keys and
    // values are then read once, not once per head
    a.pack = group > 1 && (int64_t)a.Lq * group <= 128 && xattn::lut_bytes(a, axes, group) <= 16384 ? group : 1;
    a.row_tiles = camli_divup(a.pack * a.Lq, 128);
    a.few = !training && (int64_t)a.pack * a.Lq <= 32;
    const int tile = a.few ? 32 : tile_rows(a, type);
    // few rows: a piece is shared by four waves; 512 workgroups fill the chip and leave half the parts to join (token cases above the kernel)
    split_stream(a, (int64_t)a.row_tiles * (a.H / a.pack) * a.B, camli_divup(a.Lk, tile), tile, a.few ? 512 : 1024, a.few ? 512 : type == CAMLI_F32 ? 128 : 256);
}

int dq_waves(const Args& a, int axes, bool table) { return table && axes == 1 && a.rb.buckets > 64 ? 2 : 4; }

void plan_dq(Args& a, int type, int axes, bool table) {
    a.pack = 1;
    a.row_tiles = camli_divup(a.Lq, 32 * dq_waves(a, axes, table));
    const int tile = xattn::dq_tile_rows(camli_type_size(type), padded(a.D), table);
    split_stream(a, (int64_t)a.row_tiles * a.H * a.B, camli_divup(a.Lk, tile), tile, 1024, type == CAMLI_F32 || table ? 128 : 256);
    a.parts = a.B * a.row_tiles * a.splits;
}

void plan_dkdv(Args& a, int type) {
    a.pack = 1;
    a.row_tiles = camli_divup(a.Lk, 128);
    const int tile = tile_rows(a, type);
    split_stream(a, (int64_t)a.row_tiles * a.Hk * a.B, camli_divup(a.Lq, tile) * (a.H / a.Hk), tile, 1024, type == CAMLI_F32 ? 128 : 256);
}

bool operand_ok(const void* p, const int64_t* stride, int size) {
    if (!p || ((uintptr_t)p & 15)) return false;
    for (int i = 0; i < 3; ++i)
        if (stride[i] < 0 || (stride[i] * size) & 15) return false;
    return stride[1] < (1 << 23);       // a thread's place in a tile of 64 rows is a 32-bit byte offset
}

// false (with the error set) for anything the kernels do not take
bool make_args(Args& a, const camli_attention* d, const char* who) {
    if (!d) { camli_set_error("%s: null descriptor", who); return false; }
    if (d->type < 0 || d->type > 2 || d->B < 1 || d->Hk < 1 || d->H < d->Hk || d->H % d->Hk != 0 || d->Lq < 1 || d->Lk < 1 || d->D < 8 || d->D > 128 ||
        d->D % 8 != 0 || !(d->scale >= 1e-15f) || !(d->scale <= 1e15f)) {
        camli_set_error("%s: need type 0..2, B, Lq, Lk >= 1, H a multiple of Hk, D a multiple of 8 up to 128, a scale from 1e-15 to 1e15 (type=%d B=%d H=%d Hk=%d Lq=%d Lk=%d D=%d scale=%g)",
                        who, d->type, d->B, d->H, d->Hk, d->Lq, d->Lk, d->D, (double)d->scale);
        return false;
    }
    const int size = camli_type_size(d->type);
    // a launch has fewer than 2^32 threads: 2^24 workgroups of 256
    if ((int64_t)d->B * d->H * camli_divup(d->Lq > INT32_MAX - 256 ? 0 : d->Lq, 32) >= (1 << 24) || (int64_t)d->B * d->Hk * camli_divup(d->Lk > INT32_MAX - 256 ? 0 : d->Lk, 128) >= (1 << 24) ||
        (int64_t)camli_divup(d->Lq > INT32_MAX - 256 ? 0 : d->Lq, 32) * (d->H / d->Hk) >= (1 << 24) || (int64_t)d->H * d->D >= (1 << 23) || d->Lq > INT32_MAX - 256 || d->Lk > INT32_MAX - 256) {
        camli_set_error("%s: B * H * Lq / 32, B * Hk * Lk / 128 (at most 2^24) or H * D (2^23) too large", who);
        return false;
    }
    if (!operand_ok(d->q, d->q_stride, size) || !operand_ok(d->k, d->k_stride, size) || !operand_ok(d->v, d->v_stride, size)) {
        camli_set_error("%s: q, k, v need 16-byte aligned addresses and non-negative strides of whole 16 bytes, row strides below 2^23 elements", who);
        return false;
    }
    a = Args{};
    a.q = d->q; a.k = d->k; a.v = d->v;
    a.qs = {d->q_stride[0], d->q_stride[1], d->q_stride[2]};
    a.ks = {d->k_stride[0], d->k_stride[1], d->k_stride[2]};
    a.vs = {d->v_stride[0], d->v_stride[1], d->v_stride[2]};
    a.lengths = d->kv_lengths;
    a.mask = d->key_mask;
    a.mask_bs = d->key_mask_batch_stride;
    a.B = d->B; a.H = d->H; a.Hk = d->Hk; a.Lq = d->Lq; a.Lk = d->Lk; a.D = d->D;
    a.scale = d->scale;
    a.scale_log2 = d->scale * xattn::LOG2E;
    if (d->bias_axes != 0 && d->H > 65535) {
        camli_set_error("%s: a position bias takes at most 65535 heads (H=%d)", who, d->H);
        return false;
    }
    if (d->bias_axes != 0 && !rel_bias_args(a.rb, who, d->bias_table, d->type, d->q_pos, d->q_pos_batch_stride, d->k_pos, d->k_pos_batch_stride,
                                            d->bias_axes, d->bias_buckets, d->bias_two_sided, d->bias_max_distance))
        return false;
    return true;
}

int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// workspace of the forward: part_o, part_lse
int64_t fwd_workspace(Args& a, char* base) {
    if (a.splits == 1) return 0;
    const int64_t rows = (int64_t)a.B * a.Lq * a.H, o = align256(4 * rows * a.D * a.splits);
    a.part_o = reinterpret_cast<float*>(base);
    a.part_lse = reinterpret_cast<float*>(base + o);
    return o + align256(8 * rows * a.splits);
}

struct BwdPlan {
    Args dq, dkdv;
    int64_t bytes;
};

// workspace of the backward: delta, which rows are far, then the parts of dq, of the table, of dk and dv
BwdPlan plan_bwd(const Args& a, const camli_attention* d, bool table, char* base) {
    BwdPlan p{a, a, 0};
    plan_dq(p.dq, d->type, d->bias_axes, table);
    plan_dkdv(p.dkdv, d->type);
    const int64_t rows = (int64_t)a.B * a.H * a.Lq;
    p.dq.delta = p.dkdv.delta = reinterpret_cast<float*>(base);
    int64_t end = align256(4 * rows);
    p.dq.row_groups = p.dkdv.row_groups = p.dq.row_tiles * dq_waves(p.dq, d->bias_axes, table);
    p.dq.far_rows = p.dkdv.far_rows = reinterpret_cast<int*>(base + end);
    end += align256((int64_t)4 * a.B * a.H * p.dq.row_groups);
    if (d->type == CAMLI_F16) {
        p.dq.go_l1 = p.dkdv.go_l1 = reinterpret_cast<float*>(base + end);
        end += align256(4 * rows);
        p.dq.v_chunks = p.dkdv.v_chunks = xattn::v_chunks(a);
        p.dq.v_max = p.dkdv.v_max = reinterpret_cast<float*>(base + end);
        end += align256((int64_t)4 * a.B * a.Hk * p.dq.v_chunks);
    }
    if (p.dq.splits > 1) {
        p.dq.part_o = reinterpret_cast<float*>(base + end);
        end += align256(4 * rows * a.D * p.dq.splits);
    }
    if (table) {
        p.dq.part_table = reinterpret_cast<float*>(base + end);
        end += align256((int64_t)4 * a.H * p.dq.parts * d->bias_axes * d->bias_buckets);
    }
    if (p.dkdv.splits > 1) {
        const int64_t n = align256((int64_t)4 * a.B * a.Lk * a.Hk * a.D * p.dkdv.splits);
        p.dkdv.part_dk = reinterpret_cast<float*>(base + end);
        p.dkdv.part_dv = reinterpret_cast<float*>(base + end + n);
        end += 2 * n;
    }
    p.bytes = end;
    return p;
}

}  // namespace

extern "C" int64_t camli_cross_attention_fwd_workspace_bytes(const camli_attention* d, int training) {
    Args a;
    if (!make_args(a, d, "camli_cross_attention_fwd_workspace_bytes")) return CAMLI_EINVAL;
    plan_fwd(a, d->type, d->bias_axes, training != 0);
    return fwd_workspace(a, nullptr);
}

extern "C" int camli_cross_attention_fwd(const camli_attention* d, void* out, float* out_f32, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
    Args a;
    if (!make_args(a, d, "camli_cross_attention_fwd")) return CAMLI_EINVAL;
    plan_fwd(a, d->type, d->bias_axes, lse != nullptr);
    const int64_t need = fwd_workspace(a, static_cast<char*>(workspace));
    const bool two = lse && d->type != CAMLI_F32;
    if (!out || (((uintptr_t)out | (uintptr_t)out_f32) & 15) || (two && !out_f32) || (need > 0 && (!workspace || ((uintptr_t)workspace & 15) || workspace_bytes < need))) {
        camli_set_error("camli_cross_attention_fwd: output or workspace missing, unaligned or too small (%lld bytes needed)", (long long)need);
        return CAMLI_EINVAL;
    }
    a.out = out;
    a.out_f32 = two ? out_f32 : nullptr;
    a.lse = lse;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (d->type == CAMLI_F32) return xattn::Launch<float>::fwd(a, d->bias_axes, s);
    if (d->type == CAMLI_BF16) return xattn::Launch<__bf16>::fwd(a, d->bias_axes, s);
    return xattn::Launch<_Float16>::fwd(a, d->bias_axes, s);
}

extern "C" int64_t camli_cross_attention_bwd_workspace_bytes(const camli_attention* d, int table_gradient) {
    Args a;
    if (!make_args(a, d, "camli_cross_attention_bwd_workspace_bytes")) return CAMLI_EINVAL;
    return plan_bwd(a, d, table_gradient != 0 && d->bias_axes != 0, nullptr).bytes;
}

extern "C" int camli_cross_attention_bwd(const camli_attention* d, const float* out_f32, const void* gout, const float* lse, void* gq, void* gk,
                                         void* gv, void* gtable, void* workspace, int64_t workspace_bytes, void* stream) {
    Args a;
    if (!make_args(a, d, "camli_cross_attention_bwd")) return CAMLI_EINVAL;
    if (gtable && d->bias_axes == 0) { camli_set_error("camli_cross_attention_bwd: a table gradient without a table"); return CAMLI_EINVAL; }
    BwdPlan p = plan_bwd(a, d, gtable != nullptr, static_cast<char*>(workspace));
    if (!out_f32 || !gout || !lse || (gk == nullptr) != (gv == nullptr) || !workspace || workspace_bytes < p.bytes ||
        (((uintptr_t)out_f32 | (uintptr_t)gout | (uintptr_t)gq | (uintptr_t)gk | (uintptr_t)gv | (uintptr_t)workspace) & 15)) {
        camli_set_error("camli_cross_attention_bwd: an operand is missing or not 16-byte aligned, or the workspace is too small (%lld bytes needed)", (long long)p.bytes);
        return CAMLI_EINVAL;
    }
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int axes = d->bias_axes, waves = dq_waves(p.dq, axes, gtable != nullptr);
    p.dq.o = out_f32;
    p.dq.go = p.dkdv.go = gout;
    p.dq.lse = p.dkdv.lse = const_cast<float*>(lse);
    p.dq.dq = gq;
    p.dkdv.dk = gk;
    p.dkdv.dv = gv;
    if (d->type == CAMLI_F16) {
        const int rc = xattn::Launch<_Float16>::values(p.dq, s);
        if (rc != CAMLI_OK) return rc;
    }
    int rc = d->type == CAMLI_F32 ? xattn::Launch<float>::dq(p.dq, axes, waves, s)
             : d->type == CAMLI_BF16 ? xattn::Launch<__bf16>::dq(p.dq, axes, waves, s) : xattn::Launch<_Float16>::dq(p.dq, axes, waves, s);
    if (rc != CAMLI_OK) return rc;
    if (gk) {
        rc = d->type == CAMLI_F32 ? xattn::Launch<float>::dkdv(p.dkdv, axes, s)
             : d->type == CAMLI_BF16 ? xattn::Launch<__bf16>::dkdv(p.dkdv, axes, s) : xattn::Launch<_Float16>::dkdv(p.dkdv, axes, s);
        if (rc != CAMLI_OK) return rc;
    }
    rc = d->type == CAMLI_F32 ? xattn::Launch<float>::far(p.dq, p.dkdv, axes, waves, s)
         : d->type == CAMLI_BF16 ? xattn::Launch<__bf16>::far(p.dq, p.dkdv, axes, waves, s) : xattn::Launch<_Float16>::far(p.dq, p.dkdv, axes, waves, s);
    if (rc != CAMLI_OK) return rc;
    if (gtable) {
        rc = rel_bias_join(p.dq.part_table, gtable, d->type, a.H, axes * d->bias_buckets, p.dq.parts, "camli_cross_attention_bwd", s);
        if (rc != CAMLI_OK) return rc;
    }
    xattn::SumJobs jobs;
    int n = 0;
    if (gq && p.dq.splits > 1) jobs.job[n++] = {p.dq.part_o, gq, (int64_t)a.B * a.Lq * a.H * a.D, p.dq.splits};
    if (gk && p.dkdv.splits > 1) {
        jobs.job[n++] = {p.dkdv.part_dk, gk, (int64_t)a.B * a.Lk * a.Hk * a.D, p.dkdv.splits};
        jobs.job[n++] = {p.dkdv.part_dv, gv, (int64_t)a.B * a.Lk * a.Hk * a.D, p.dkdv.splits};
    }
    if (n == 0) return CAMLI_OK;
    if (d->type == CAMLI_F32) return xattn::Launch<float>::sum(jobs, n, s);
    if (d->type == CAMLI_BF16) return xattn::Launch<__bf16>::sum(jobs, n, s);
    return xattn::Launch<_Float16>::sum(jobs, n, s);
}
