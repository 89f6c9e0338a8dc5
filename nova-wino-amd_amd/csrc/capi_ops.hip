// C-ABI of the operators around the convolutions (include/nova_winograd.h):
// group norm and attention. No handle: the caller names the stream and owns
// the workspace. Argument checks only; the work is in group_norm.hip and
// attention_*.hip.
#include <atomic>
#include <climits>
#include <cmath>

#include "../../include/nova_winograd.h"
#include "nova_internal.h"

namespace nova {

namespace {

bool hip_ok(hipError_t e, const char* what) {
    if (e == hipSuccess) return true;
    set_error(e == hipErrorOutOfMemory ? kErrOutOfMemory : kErrHip, "%s: %s", what,
              hipGetErrorString(e));
    return false;
}

// Compute units of the current device (256 where it cannot be asked).
int compute_units() {
    static std::atomic<int> known[64];
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) == hipSuccess && dev >= 0 && dev < 64) {
        cus = known[dev].load(std::memory_order_relaxed);
        if (cus > 0) return cus;
        if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) ==
                hipSuccess &&
            cus > 0) {
            known[dev].store(cus, std::memory_order_relaxed);
            return cus;
        }
    }
    (void)hipGetLastError();
    return 256;
}

// a * b, or -1 where it passes 2^62 (a, b >= 0; -1 stays -1).
int64_t times(int64_t a, int64_t b) {
    if (a < 0 || b < 0) return -1;
    if (b != 0 && a > (INT64_C(1) << 62) / b) return -1;
    return a * b;
}

bool workspace_ok(const char* fn, const void* ws, long long have, int64_t need) {
    if (need <= 0) return true;
    if (ws != nullptr && have >= need && reinterpret_cast<uintptr_t>(ws) % 16 == 0) return true;
    set_error(kErrWorkspace, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", fn,
              (long long)need, ws ? have : 0ll);
    return false;
}

bool aligned(const void* p, size_t size) { return reinterpret_cast<uintptr_t>(p) % size == 0; }
bool aligned(const void* p, const GroupNorm& g) { return aligned(p, g.dtype == kF32 ? 4 : 2); }

bool group_norm_args(const char* fn, const nova_group_norm_t* p, GroupNorm* g) {
    if (p == nullptr) {
        set_error(kErrInvalidArgument, "%s: null arguments", fn);
        return false;
    }
    if (p->dtype < 0 || p->dtype > 2 || p->param_dtype < 0 || p->param_dtype > 2) {
        set_error(kErrInvalidArgument, "%s: unknown type (%d, parameters %d)", fn, p->dtype,
                  p->param_dtype);
        return false;
    }
    if (p->batch < 0 || p->channels < 1 || p->groups < 1 || p->channels % p->groups != 0 ||
        p->pixels < 0 || (p->channels_last != 0 && p->channels_last != 1) ||
        (p->silu != 0 && p->silu != 1) || !(p->eps >= 0.0f) || !std::isfinite(p->eps)) {
        set_error(kErrInvalidArgument,
                  "%s: bad shape or option (batch %d, channels %d, groups %d, pixels %lld, eps %g)",
                  fn, p->batch, p->channels, p->groups, (long long)p->pixels, (double)p->eps);
        return false;
    }
    const int64_t n = times(times(p->batch, p->channels), p->pixels);
    // the kernels' walks over an image's pixels step past its end by less than 2^20
    if (n < 0 || n > (INT64_C(1) << 40) || p->pixels > INT_MAX - (1 << 20) ||
        (int64_t)p->batch * p->groups > (1 << 30) || (int64_t)p->batch * p->channels > (1 << 30)) {
        set_error(kErrInvalidArgument, "%s: shape exceeds launch limits", fn);
        return false;
    }
    const size_t size = p->dtype == 2 ? 4 : 2;
    if (n > 0 && (p->x == nullptr || reinterpret_cast<uintptr_t>(p->x) % size != 0)) {
        set_error(kErrInvalidArgument, "%s: null or misaligned input", fn);
        return false;
    }
    *g = GroupNorm{p->x,     p->weight, p->bias,          p->dtype, p->param_dtype, p->batch,
                   p->channels, p->groups, p->pixels, p->channels_last, p->silu, p->eps};
    return true;
}

// Whether every launch of the call has fewer than 2^32 threads, which is what a
// grid takes. Below 2^21 images times channels none comes near that many.
bool group_norm_fits(const char* fn, const GroupNorm& g, bool backward, int cus) {
    if ((int64_t)g.B * g.C < (1 << 21) ||
        group_norm_launch(g, backward, cus).threads < (INT64_C(1) << 32))
        return true;
    set_error(kErrInvalidArgument, "%s: shape exceeds launch limits", fn);
    return false;
}

bool attention_args(const char* fn, const nova_attention_t* p, Attention* a) {
    if (p == nullptr) {
        set_error(kErrInvalidArgument, "%s: null arguments", fn);
        return false;
    }
    if (p->dtype != 0 && p->dtype != 1) {
        set_error(kErrInvalidArgument, "%s: type must be float16 (0) or bfloat16 (1)", fn);
        return false;
    }
    if (p->batch < 0 || (p->kv_batch != p->batch && p->kv_batch != 1) || p->queries < 0 ||
        p->keys < 0 || p->heads < 1 || p->kv_heads < 1 || p->heads % p->kv_heads != 0 ||
        p->head_dim < 1 || p->head_dim > 256 || !std::isfinite(p->scale)) {
        set_error(kErrInvalidArgument,
                  "%s: bad shape (batch %d / %d, queries %d, keys %d, heads %d / %d, head_dim %d)",
                  fn, p->batch, p->kv_batch, p->queries, p->keys, p->heads, p->kv_heads,
                  p->head_dim);
        return false;
    }
    // A head of a sequence takes a workgroup of 256 threads, or one for each 128
    // of its rows (or keys): fewer than 2^24 heads in all, and 2^29 rows, keep
    // every launch below 2^32 threads.
    const int64_t rows = times(times(p->batch, p->heads), p->queries);
    const int64_t keys = times(times(p->kv_batch, p->kv_heads), p->keys);
    if (rows < 0 || keys < 0 || times(rows, p->head_dim) > (INT64_C(1) << 36) ||
        times(keys, p->head_dim) > (INT64_C(1) << 36) || rows > (1 << 29) || keys > (1 << 29) ||
        p->queries > (1 << 28) || p->keys > (1 << 28) ||
        (int64_t)p->batch * p->heads >= (1 << 24) ||
        (int64_t)p->kv_batch * p->kv_heads >= (1 << 24)) {
        set_error(kErrInvalidArgument, "%s: shape exceeds launch limits", fn);
        return false;
    }
    if (rows > 0 && (p->q == nullptr || reinterpret_cast<uintptr_t>(p->q) % 2 != 0)) {
        set_error(kErrInvalidArgument, "%s: null or misaligned queries", fn);
        return false;
    }
    if (keys > 0 && (p->k == nullptr || p->v == nullptr ||
                     (reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) % 2)) {
        set_error(kErrInvalidArgument, "%s: null or misaligned keys or values", fn);
        return false;
    }
    if (p->key_mask != nullptr && p->mask_stride < 0) {
        set_error(kErrInvalidArgument, "%s: negative mask stride", fn);
        return false;
    }
    *a = Attention{};
    a->q = static_cast<const uint16_t*>(p->q);
    a->k = static_cast<const uint16_t*>(p->k);
    a->v = static_cast<const uint16_t*>(p->v);
    a->mask = p->key_mask;
    for (int i = 0; i < 3; i++) {
        a->qs[i] = p->q_strides[i];
        a->ks[i] = p->k_strides[i];
        a->vs[i] = p->v_strides[i];
    }
    a->mask_stride = p->mask_stride;
    a->B = p->batch;
    a->Bk = p->kv_batch;
    a->Lq = p->queries;
    a->Lk = p->keys;
    a->H = p->heads;
    a->KV = p->kv_heads;
    a->D = p->head_dim;
    a->bf16 = p->dtype;
    a->scale = p->scale;
    return true;
}

}  // namespace

}  // namespace nova

using namespace nova;

extern "C" {

long long nova_group_norm_workspace_bytes(const nova_group_norm_t* p, int backward) {
    GroupNorm g;
    const char* fn = "nova_group_norm_workspace_bytes";
    if (!group_norm_args(fn, p, &g)) return -1;
    const int cus = compute_units();
    if (!group_norm_fits(fn, g, backward != 0, cus)) return -1;
    return backward ? group_norm_bwd_ws(g, cus) : group_norm_ws(g, cus);
}

void nova_group_norm(const nova_group_norm_t* p, void* d_y, float* d_mean, float* d_rstd,
                     void* d_workspace, long long workspace_bytes, void* stream) {
    const char* fn = "nova_group_norm";
    GroupNorm g;
    if (!group_norm_args(fn, p, &g)) return;
    if (g.B == 0 || g.P == 0) return;
    if (d_y == nullptr || d_mean == nullptr || d_rstd == nullptr) {
        set_error(kErrInvalidArgument, "%s: null output", fn);
        return;
    }
    if (!aligned(d_y, g) || !aligned(d_mean, 4) || !aligned(d_rstd, 4)) {
        set_error(kErrInvalidArgument, "%s: misaligned output", fn);
        return;
    }
    const int cus = compute_units();
    if (!group_norm_fits(fn, g, false, cus)) return;
    if (!workspace_ok(fn, d_workspace, workspace_bytes, group_norm_ws(g, cus))) return;
    hip_ok(launch_group_norm(g, d_y, d_mean, d_rstd, d_workspace, cus,
                             static_cast<hipStream_t>(stream)),
           fn);
}

void nova_group_norm_backward(const nova_group_norm_t* p, const void* d_grad_y,
                              const float* d_mean, const float* d_rstd, void* d_grad_x,
                              void* d_grad_weight, void* d_grad_bias, void* d_workspace,
                              long long workspace_bytes, void* stream) {
    const char* fn = "nova_group_norm_backward";
    GroupNorm g;
    if (!group_norm_args(fn, p, &g)) return;
    if ((d_grad_weight == nullptr) != (d_grad_bias == nullptr)) {
        set_error(kErrInvalidArgument, "%s: weight and bias gradients are given together", fn);
        return;
    }
    const bool none = g.B == 0 || g.P == 0;
    if (!none && (d_grad_y == nullptr || d_mean == nullptr || d_rstd == nullptr ||
                  d_grad_x == nullptr)) {
        set_error(kErrInvalidArgument, "%s: null argument", fn);
        return;
    }
    if (!none && (!aligned(d_grad_y, g) || !aligned(d_grad_x, g) || !aligned(d_mean, 4) ||
                  !aligned(d_rstd, 4))) {
        set_error(kErrInvalidArgument, "%s: misaligned argument", fn);
        return;
    }
    const int cus = compute_units();
    if (!group_norm_fits(fn, g, true, cus)) return;
    if (!none &&
        !workspace_ok(fn, d_workspace, workspace_bytes, group_norm_bwd_ws(g, cus)))
        return;
    hip_ok(launch_group_norm_bwd(g, d_grad_y, d_mean, d_rstd, d_grad_x, d_grad_weight,
                                 d_grad_bias, d_workspace, cus, static_cast<hipStream_t>(stream)),
           fn);
}

long long nova_cross_attention_workspace_bytes(const nova_attention_t* p, int backward) {
    Attention a;
    if (!attention_args("nova_cross_attention_workspace_bytes", p, &a)) return -1;
    const int cus = compute_units();
    return backward ? attention_bwd_plan(a, cus).ws_bytes : attention_plan(a, cus).ws_bytes;
}

int nova_cross_attention_uses_rest(const nova_attention_t* p) {
    Attention a;
    if (!attention_args("nova_cross_attention_uses_rest", p, &a)) return -1;
    return attention_uses_rest(a);
}

void nova_cross_attention(const nova_attention_t* p, void* d_out, void* d_rest, float* d_lse,
                          void* d_workspace, long long workspace_bytes, void* stream) {
    const char* fn = "nova_cross_attention";
    Attention a;
    if (!attention_args(fn, p, &a)) return;
    if (a.B == 0 || a.Lq == 0) return;
    if (d_out == nullptr || !aligned(d_out, 16) || !aligned(d_rest, 16) || !aligned(d_lse, 4)) {
        set_error(kErrInvalidArgument, "%s: an output is null or not 16-byte aligned", fn);
        return;
    }
    const AttentionPlan plan = attention_plan(a, compute_units());
    if (!workspace_ok(fn, d_workspace, workspace_bytes, plan.ws_bytes)) return;
    hip_ok(launch_attention(a, plan, static_cast<uint16_t*>(d_out), static_cast<uint16_t*>(d_rest),
                            d_lse, d_workspace, static_cast<hipStream_t>(stream)),
           fn);
}

void nova_cross_attention_backward(const nova_attention_t* p, const void* d_out,
                                   const void* d_rest, const float* d_lse, const void* d_grad_out, void* d_grad_q,
                                   void* d_grad_k, void* d_grad_v, void* d_workspace,
                                   long long workspace_bytes, void* stream) {
    const char* fn = "nova_cross_attention_backward";
    Attention a;
    if (!attention_args(fn, p, &a)) return;
    const bool rows = a.B > 0 && a.Lq > 0, keys = a.Bk > 0 && a.Lk > 0;
    if ((rows && (d_out == nullptr || d_lse == nullptr || d_grad_out == nullptr ||
                  d_grad_q == nullptr || !aligned(d_out, 2) || !aligned(d_rest, 2) ||
                  !aligned(d_lse, 4) || !aligned(d_grad_out, 2) || !aligned(d_grad_q, 16))) ||
        (keys && (d_grad_k == nullptr || d_grad_v == nullptr || !aligned(d_grad_k, 16) ||
                  !aligned(d_grad_v, 16)))) {
        set_error(kErrInvalidArgument, "%s: null or misaligned argument", fn);
        return;
    }
    if (!rows && !keys) return;
    const AttentionBwdPlan plan = attention_bwd_plan(a, compute_units());
    if (!workspace_ok(fn, d_workspace, workspace_bytes, plan.ws_bytes)) return;
    hip_ok(launch_attention_bwd(a, plan, static_cast<const uint16_t*>(d_out),
                                static_cast<const uint16_t*>(d_rest), d_lse,
                                static_cast<const uint16_t*>(d_grad_out),
                                static_cast<uint16_t*>(d_grad_q), static_cast<uint16_t*>(d_grad_k),
                                static_cast<uint16_t*>(d_grad_v), d_workspace,
                                static_cast<hipStream_t>(stream)),
           fn);
}

}  // extern "C"
