// C entries of attention under a described mask: plan, checks of arguments, choice of the kernel.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <initializer_list>
#include <new>
#include <string>
#include <utility>

#include "attention.cuh"
#include "device_guard.hpp"
#include "engine_internal.hpp"
#include "sddmm_b200.h"
#include "tc_utils.cuh"

struct sddmm_attention_s {
    sddmm_handle_s *h = nullptr;
    AttentionParams p{};
    ForwardPlan few{}, prompt{};  // of which the quicker one is taken
    bool by_few = false, tensor_cores = false;
    Parts parts = ONE_PART;
    const char *last_kernel = "none";
};

namespace {

constexpr int64_t MAX_ROWS = 1 << 29;
constexpr int MAX_WINDOW = (1 << 30) - 1;  // more than any distance
constexpr int MAX_HEAD_DIM = 128;

int bad(sddmm_handle_s *h, const char *why)
{
    h->last_error = why;
    return SDDMM_INVALID_ARG;
}

// An array of the call: in memory of the handle's GPU, aligned to its elements.  rows 0: it may be anything.
int check_array(sddmm_handle_s *h, const sddmm_head_array *a, const char *name, int dtype, int head_dim, int heads, int64_t rows, bool written,
                HeadArray *out)
{
    const size_t size = dtype == SDDMM_F32 ? 4 : 2;
    if (!a) {
        h->last_error = std::string(name) + " is missing";
        return SDDMM_INVALID_ARG;
    }
    *out = HeadArray{a->data, a->row_stride, a->head_stride};
    if (rows == 0) return SDDMM_OK;
    if (!on_device(a->data, h->device) || (uintptr_t)a->data % size != 0) {
        h->last_error = std::string(name) + " must be device memory of the handle's GPU, aligned to its elements";
        return SDDMM_INVALID_ARG;
    }
    if (a->row_stride < 0 || a->head_stride < 0) {
        h->last_error = std::string(name) + " has a negative stride";
        return SDDMM_INVALID_ARG;
    }
    if (written && !(strides_apart(a->head_stride, heads, a->row_stride, rows, head_dim))) {
        h->last_error = std::string(name) + " is written, and its strides let entries overlap";
        return SDDMM_INVALID_ARG;
    }
    return SDDMM_OK;
}

// Whether an array that is written starts where one of `others` does (arrays without rows are nobody's).
bool same_start(const HeadArray &w, int64_t rows, std::initializer_list<std::pair<const HeadArray *, int64_t>> others)
{
    for (const auto &o : others)
        if (rows > 0 && o.second > 0 && w.data == o.first->data) return true;
    return false;
}
constexpr const char *OVERLAP = "an array that is written is also read, or written as another";
// Of offsets, lengths, slopes and lse: 32-bit values in memory of the handle's GPU.
bool words_on_device(const void *p, int device) { return (uintptr_t)p % 4 == 0 && on_device(p, device); }

// delta of the backward pass, first in its workspace, and in fp16 what its tiles of dO hold at most
int64_t delta_bytes(const AttentionParams &p) { return ((int64_t)sizeof(float) * p.q_heads * p.q_rows + 15) / 16 * 16; }
int64_t most_bytes(const AttentionParams &p) { return p.dtype == SDDMM_F16 ? ((int64_t)sizeof(float) * p.q_heads * most_tiles(p) + 15) / 16 * 16 : 0; }

bool capturing(cudaStream_t s)
{
    cudaStreamCaptureStatus c = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(s, &c) == cudaSuccess && c != cudaStreamCaptureStatusNone;
}

int finish(sddmm_attention_s *a, cudaError_t e, const char *name, int launches, uint32_t flags)
{
    sddmm_handle_s *h = a->h;
    if (e == cudaSuccess) {
        a->last_kernel = name;
        h->n_launches += launches;
        if (flags & SDDMM_FLAG_ASYNC) return SDDMM_OK;
        e = cudaStreamSynchronize(h->stream);
        if (e == cudaSuccess) return device_status(h);
    }
    h->last_error = std::string(name) + ": " + cudaGetErrorString(e);
    (void)cudaGetLastError();
    return SDDMM_CUDA_ERROR;
}

}  // namespace

int sddmm_attention_plan(sddmm_handle_t h, const sddmm_attention_desc *d, sddmm_attention_t *out)
{
    if (!h || !out) return SDDMM_INVALID_ARG;
    *out = nullptr;
    if (!d) return bad(h, "no description");
    if (d->dtype != SDDMM_F32 && d->dtype != SDDMM_F16 && d->dtype != SDDMM_BF16) return bad(h, "unknown dtype");
    if (d->head_dim < 8 || d->head_dim > MAX_HEAD_DIM || d->head_dim % 8) {
        h->last_error = "head_dim must be a multiple of 8 from 8 to 128";
        return SDDMM_K_UNSUPPORTED;
    }
    if (d->q_heads < 1 || d->kv_heads < 1 || d->q_heads % d->kv_heads) return bad(h, "q_heads must be a multiple of kv_heads");
    if (d->n_seqs < 0 || d->max_q < 0 || d->max_k < 0) return bad(h, "negative size");
    if (d->q_rows < 0 || d->q_rows > MAX_ROWS || d->k_rows < 0 || d->k_rows > MAX_ROWS) return bad(h, "q_rows and k_rows go from 0 to 2^29");
    if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return bad(h, "scale must be positive and finite");
    if (!(d->softcap >= 0.f) || !std::isfinite(d->softcap)) return bad(h, "softcap must be 0 (none) or positive and finite");
    if (d->window_left < -1 || d->window_right < -1) return bad(h, "a window's side is -1 (no limit), 0 or positive");
    DeviceGuard guard(h->device);
    if (d->n_seqs > 0 && !words_on_device(d->q_offsets, h->device)) return bad(h, "q_offsets must be aligned device memory of the handle's GPU");
    if (d->k_len && !d->k_offsets) return bad(h, "k_len goes with k_offsets");
    const void *more[] = {d->k_offsets, d->k_len, d->prefix, d->slopes};
    for (const void *x : more)
        if (x && d->n_seqs > 0 && !words_on_device(x, h->device)) return bad(h, "k_offsets, k_len, prefix and slopes must be aligned device memory of the handle's GPU");
    AttentionParams p{};
    p.dtype = d->dtype;
    p.head_dim = d->head_dim;
    p.q_heads = d->q_heads;
    p.kv_heads = d->kv_heads;
    p.group = d->q_heads / d->kv_heads;
    p.n_seqs = d->n_seqs;
    p.q_rows = d->q_rows;
    p.k_rows = d->k_offsets ? d->k_rows : d->q_rows;
    if (!d->k_offsets && d->k_rows != d->q_rows) return bad(h, "without k_offsets K has the rows of Q");
    p.max_q = (int)(d->max_q < d->q_rows ? d->max_q : d->q_rows);
    p.max_k = (int)(d->max_k < p.k_rows ? d->max_k : p.k_rows);
    p.scale = d->scale;
    p.cap = d->softcap;
    p.window.left = d->window_left < MAX_WINDOW ? d->window_left : MAX_WINDOW;
    p.window.right = d->window_right < MAX_WINDOW ? d->window_right : MAX_WINDOW;
    p.q_offsets = d->q_offsets;
    p.k_offsets = d->k_offsets;
    p.k_len = d->k_len;
    p.prefix = d->prefix;
    p.slopes = d->slopes;
    p.status = h->d_status;
    if ((most_blocks(p.q_rows, p.n_seqs, p.max_q, 16) + 1) * p.q_heads > INT_MAX || (most_blocks(p.k_rows, p.n_seqs, p.max_k, 64) + 1) * p.q_heads > INT_MAX)
        return bad(h, "too many heads and rows for one launch");
    // (a cap that is not within a factor of a million of the scale: its tanh, whose factors might leave fp32's range here, is left to the
    // general kernels' own; a scale beyond that: likewise)
    const float of_cap = p.cap == 0.f ? 1.f : p.scale / p.cap;
    const bool reach = of_cap >= tc::TANH_LEAST && of_cap <= tc::TANH_MOST;
    p.of_cap = reach ? of_cap : 1.f;
    p.pre = reach ? 1.f : of_cap;
    sddmm_attention_s *a = new (std::nothrow) sddmm_attention_s;
    if (!a) return SDDMM_OUT_OF_MEMORY;
    a->h = h;
    a->p = p;
    a->tensor_cores = p.dtype != SDDMM_F32 && of_cap >= 1e-6f && of_cap <= 1e6f && p.scale <= 1e6f;
    if (a->tensor_cores) {
        a->few = plan_attention_few_tc(p, h->sm_count);
        a->prompt = plan_attention_forward_tc(p, h->sm_count);
        a->by_few = a->few.n_splits > 0 && a->few.us < a->prompt.us;
    }
    if (!a->tensor_cores) a->prompt = plan_attention_forward_general(p, h->sm_count);
    if (p.dtype == SDDMM_F32) {
        a->few = plan_attention_few_f32(p, h->sm_count);
        a->by_few = a->few.n_splits > 0 && a->few.us < a->prompt.us;
    }
    a->parts = p.dtype == SDDMM_F32 ? plan_attention_parts(p, 64, 4, h->sm_count) : plan_attention_parts(p, 128, 1, h->sm_count);
    *out = a;
    return SDDMM_OK;
}

int sddmm_attention_destroy(sddmm_attention_t a)
{
    delete a;
    return SDDMM_OK;
}

int sddmm_attention_workspace(sddmm_attention_t a, int backward, int64_t *bytes)
{
    if (!a || !bytes) return SDDMM_INVALID_ARG;
    *bytes = backward ? delta_bytes(a->p) + most_bytes(a->p) + a->parts.bytes : a->by_few ? a->few.bytes : a->prompt.bytes;
    return SDDMM_OK;
}

int sddmm_attention_forward(sddmm_attention_t a, const sddmm_head_array *Q, const sddmm_head_array *K, const sddmm_head_array *V,
                            const sddmm_head_array *O, float *lse, void *workspace, int64_t workspace_bytes, uint32_t flags)
{
    if (!a) return SDDMM_INVALID_ARG;
    sddmm_handle_s *h = a->h;
    if (flags & ~(uint32_t)SDDMM_FLAG_ASYNC) return bad(h, "unknown flag");
    AttentionParams p = a->p;
    DeviceGuard guard(h->device);
    int st;
    if ((st = check_array(h, Q, "Q", p.dtype, p.head_dim, p.q_heads, p.q_rows, false, &p.q))) return st;
    if ((st = check_array(h, K, "K", p.dtype, p.head_dim, p.kv_heads, p.k_rows, false, &p.k))) return st;
    if ((st = check_array(h, V, "V", p.dtype, p.head_dim, p.kv_heads, p.k_rows, false, &p.v))) return st;
    if ((st = check_array(h, O, "O", p.dtype, p.head_dim, p.q_heads, p.q_rows, true, &p.o))) return st;
    if (same_start(p.o, p.q_rows, {{&p.q, p.q_rows}, {&p.k, p.k_rows}, {&p.v, p.k_rows}})) return bad(h, OVERLAP);
    if (lse && p.q_rows > 0 && !words_on_device(lse, h->device)) return bad(h, "lse must be aligned device memory of the handle's GPU");
    p.lse = lse;
    int64_t need = 0;
    sddmm_attention_workspace(a, 0, &need);
    if (need > 0 && (workspace_bytes < need || !on_device(workspace, h->device) || (uintptr_t)workspace % 16))
        return bad(h, "workspace: sddmm_attention_workspace() bytes of device memory, 16-byte aligned");
    if (!(flags & SDDMM_FLAG_ASYNC) && capturing(h->stream)) return bad(h, "a captured call must be asynchronous");
    if (p.n_seqs == 0) return SDDMM_OK;
    // (no queries: the general kernel has one block, which looks whether the sequences agree)
    if (a->tensor_cores && p.max_q > 0) {
        bool taken = false;
        const ForwardPlan &f = a->by_few ? a->few : a->prompt;
        const cudaError_t e = a->by_few ? launch_attention_few_tc(p, f, workspace, &taken, h->stream) : launch_attention_forward_tc(p, f, workspace, &taken, h->stream);
        if (taken) return finish(a, e, a->by_few ? "attention_few_tc" : "attention_tc", f.n_splits > 1 ? 2 : 1, flags);
    }
    if (p.dtype == SDDMM_F32 && a->by_few) {
        bool taken = false;
        const cudaError_t e = launch_attention_few_f32(p, a->few, workspace, &taken, h->stream);
        if (taken) return finish(a, e, "attention_few_f32", a->few.n_splits > 1 ? 2 : 1, flags);
    }
    const ForwardPlan one{1, 1 << 30, 0, 0.}, &f = a->tensor_cores || a->by_few ? one : a->prompt;
    return finish(a, launch_attention_forward_general(p, f, workspace, h->stream), "attention_general", f.n_splits > 1 ? 2 : 1, flags);
}

int sddmm_attention_backward(sddmm_attention_t a, const sddmm_head_array *Q, const sddmm_head_array *K, const sddmm_head_array *V,
                             const sddmm_head_array *O, const float *lse, const sddmm_head_array *dO, const sddmm_head_array *dQ,
                             const sddmm_head_array *dK, const sddmm_head_array *dV, void *workspace, int64_t workspace_bytes,
                             uint32_t flags)
{
    if (!a) return SDDMM_INVALID_ARG;
    sddmm_handle_s *h = a->h;
    if (flags & ~(uint32_t)SDDMM_FLAG_ASYNC) return bad(h, "unknown flag");
    AttentionParams p = a->p;
    DeviceGuard guard(h->device);
    int st;
    if ((st = check_array(h, Q, "Q", p.dtype, p.head_dim, p.q_heads, p.q_rows, false, &p.q))) return st;
    if ((st = check_array(h, K, "K", p.dtype, p.head_dim, p.kv_heads, p.k_rows, false, &p.k))) return st;
    if ((st = check_array(h, V, "V", p.dtype, p.head_dim, p.kv_heads, p.k_rows, false, &p.v))) return st;
    if ((st = check_array(h, O, "O", p.dtype, p.head_dim, p.q_heads, p.q_rows, false, &p.o))) return st;
    if ((st = check_array(h, dO, "dO", p.dtype, p.head_dim, p.q_heads, p.q_rows, false, &p.d_o))) return st;
    if ((st = check_array(h, dQ, "dQ", p.dtype, p.head_dim, p.q_heads, p.q_rows, true, &p.dq))) return st;
    if ((st = check_array(h, dK, "dK", p.dtype, p.head_dim, p.kv_heads, p.k_rows, true, &p.dk))) return st;
    if ((st = check_array(h, dV, "dV", p.dtype, p.head_dim, p.kv_heads, p.k_rows, true, &p.dv))) return st;
    const std::initializer_list<std::pair<const HeadArray *, int64_t>> read = {{&p.q, p.q_rows}, {&p.k, p.k_rows}, {&p.v, p.k_rows}, {&p.o, p.q_rows}, {&p.d_o, p.q_rows}};
    if (same_start(p.dq, p.q_rows, read) || same_start(p.dk, p.k_rows, read) || same_start(p.dv, p.k_rows, read) ||
        same_start(p.dq, p.q_rows, {{&p.dk, p.k_rows}, {&p.dv, p.k_rows}}) || same_start(p.dk, p.k_rows, {{&p.dv, p.k_rows}}))
        return bad(h, OVERLAP);
    if (p.q_rows > 0 && !words_on_device(lse, h->device)) return bad(h, "lse must be aligned device memory of the handle's GPU");
    p.lse = const_cast<float *>(lse);
    int64_t need = 0;
    sddmm_attention_workspace(a, 1, &need);
    if (need > 0 && (workspace_bytes < need || !on_device(workspace, h->device) || (uintptr_t)workspace % 16))
        return bad(h, "workspace: sddmm_attention_workspace() bytes of device memory, 16-byte aligned");
    p.delta = static_cast<float *>(workspace);
    p.d_o_most = reinterpret_cast<float *>(static_cast<char *>(workspace) + delta_bytes(p));
    p.part_o = reinterpret_cast<float *>(static_cast<char *>(workspace) + delta_bytes(p) + most_bytes(p));
    if (!(flags & SDDMM_FLAG_ASYNC) && capturing(h->stream)) return bad(h, "a captured call must be asynchronous");
    if (p.n_seqs == 0) return SDDMM_OK;
    const bool nothing = p.max_q == 0 && p.max_k == 0;  // (as in the forward call)
    bool taken = false;
    const int launches = 2 + (a->parts.n_q > 1) + (a->parts.n_kv > 1);
    const cudaError_t e = a->tensor_cores && !nothing ? launch_attention_backward_tc(p, a->parts, &taken, h->stream) : cudaSuccess;
    if (taken) return finish(a, e, "attention_backward_tc", launches, flags);
    // (16-bit types come to the general kernels for their strides or alignment alone)
    if (p.dtype == SDDMM_F32) return finish(a, launch_attention_backward_general(p, a->parts, h->stream), "attention_backward_general", launches, flags);
    return finish(a, launch_attention_backward_general(p, ONE_PART, h->stream), "attention_backward_general", 2, flags);
}

const char *sddmm_attention_last_kernel(sddmm_attention_t a) { return a ? a->last_kernel : "none"; }
