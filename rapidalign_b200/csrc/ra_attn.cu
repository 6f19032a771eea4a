// ra_attn.cu -- host side of kernel attention (ra_attn.cuh).
#include <algorithm>

#include "ra_attn.cuh"
#include "ra_host.h"

namespace {

using namespace ra;

bool attn_ok(const ra_attn_desc *d) {
  if (d == nullptr || d->graphs < 0 || d->num_q < 0 || d->num_k < 0) return false;
  if (d->num_q > ((int64_t)1 << 31) - 256 || d->num_k > ((int64_t)1 << 31) - 256) return false;
  if (d->heads < 1 || d->kv_heads < 1 || d->heads > 4096 || d->heads % d->kv_heads) return false;
  if (std::max(d->num_q, d->num_k) * d->heads > (int64_t)1 << 32) return false;
  if (d->dim < 1 || d->dim > kAttnMaxDim || d->pos_dim < 0 || d->pos_dim > 3) return false;
  if (d->dtype < RA_F32 || d->dtype > RA_F16) return false;
  if (!(d->softcap >= 0.f) || !(d->softcap < INFINITY) || !(d->scale - d->scale == 0.f))
    return false;
  if (d->q_row < 0 || d->q_head < 0 || d->k_row < 0 || d->k_head < 0 || d->v_row < 0 ||
      d->v_head < 0)
    return false;
  if (d->max_q < 0 || d->max_k < 0 || d->max_q > d->num_q || d->max_k > d->num_k) return false;
  return d->q_tiles >= 0 && d->k_tiles >= 0 && d->status != nullptr;
}

bool inputs_ok(const ra_attn_desc *d, const ra_attn_inputs *in) {
  if (in == nullptr || (in->q_ptr == nullptr) != (in->k_ptr == nullptr)) return false;
  if (in->q_ptr != nullptr) {
    if ((d->q_tiles > 0 && in->q_tiles == nullptr) || (d->k_tiles > 0 && in->k_tiles == nullptr))
      return false;
  } else if (d->num_q != d->graphs * d->max_q || d->num_k != d->graphs * d->max_k ||
             d->q_tiles != d->graphs * ceil_div(d->max_q, (int64_t)128) ||
             d->k_tiles != d->graphs * ceil_div(d->max_k, (int64_t)128)) {
    return false;
  }
  if (d->num_q > 0 && (in->q == nullptr || d->graphs < 1)) return false;
  if (d->num_k > 0 && (in->k == nullptr || in->v == nullptr || d->graphs < 1)) return false;
  if (d->pos_dim > 0 && ((d->num_q > 0 && in->q_pos == nullptr) ||
                         (d->num_k > 0 && in->k_pos == nullptr) || in->sigma == nullptr))
    return false;
  return true;
}

AttnArgs args_of(const ra_attn_desc *d, const ra_attn_inputs *in) {
  AttnArgs a{};
  a.graphs = d->graphs, a.num_q = d->num_q, a.num_k = d->num_k;
  a.q_row = d->q_row, a.q_head = d->q_head, a.k_row = d->k_row, a.k_head = d->k_head;
  a.v_row = d->v_row, a.v_head = d->v_head;
  a.q = in->q, a.k = in->k, a.v = in->v;
  a.qs = {in->q_ptr, (const int2 *)in->q_tiles, d->max_q};
  a.ks = {in->k_ptr, (const int2 *)in->k_tiles, d->max_k};
  a.n_q_tiles = d->q_tiles, a.n_k_tiles = d->k_tiles;
  a.q_pos = d->pos_dim ? in->q_pos : nullptr, a.k_pos = d->pos_dim ? in->k_pos : nullptr;
  a.sigma = in->sigma;
  a.q_mask = in->q_mask, a.k_mask = in->k_mask;
  a.heads = d->heads, a.kv_heads = d->kv_heads, a.dim = d->dim, a.pos_dim = d->pos_dim;
  a.scale = d->scale, a.cap = d->softcap;
  a.status = d->status;
  return a;
}

struct AttnBwd {
  size_t delta, pos_q, pos_k, total;
};
AttnBwd bwd_layout(const ra_attn_desc *d) {
  AttnBwd b{};
  size_t o = 0;
  b.delta = o;
  o += align256(sizeof(float) * (size_t)d->num_q * d->heads);
  b.pos_q = o;
  if (d->pos_dim) o += align256(sizeof(float4) * (size_t)d->num_q * d->heads);
  b.pos_k = o;
  if (d->pos_dim) o += align256(sizeof(float4) * (size_t)d->num_k * d->kv_heads);
  b.total = o;
  return b;
}

unsigned grid_rows(int64_t n, int per) { return (unsigned)ceil_div(n, (int64_t)per); }

template <class T>
int forward(const AttnArgs &a, cudaStream_t st) {
  attn_row_fwd_kernel<T>
      <<<grid_rows(a.num_q * a.heads, kAttnWarps), 32 * kAttnWarps, 0, st>>>(a);
  return launched();
}

template <class T>
int backward(AttnArgs a, const ra_attn_grads *gr, char *ws, cudaStream_t st) {
  int rc;
  const int sms = sm_count();
  if (a.num_q > 0) {
    const unsigned grid =
        (unsigned)std::min<int64_t>(ceil_div(a.num_q * a.heads, (int64_t)8), (int64_t)sms * 16);
    attn_delta_kernel<T><<<grid, 256, 0, st>>>((const T *)a.dout, (const T *)a.out, a.out32,
                                               a.num_q, a.heads, a.dim, (float *)a.delta);
    if ((rc = launched())) return rc;
    if (a.dq || a.pos_q) {
      attn_row_dq_kernel<T>
          <<<grid_rows(a.num_q * a.heads, kAttnWarps), 32 * kAttnWarps, 0, st>>>(a);
      if ((rc = launched())) return rc;
    }
  }
  if (a.num_k > 0 && (a.dk || a.dv || a.pos_k)) {
    attn_row_dkv_kernel<T>
        <<<grid_rows(a.num_k * a.kv_heads, kAttnWarps), 32 * kAttnWarps, 0, st>>>(a);
    if ((rc = launched())) return rc;
  }
  if (gr->dq_pos && a.num_q > 0) {
    attn_pos_kernel<<<(unsigned)std::min<int64_t>(ceil_div(a.num_q, (int64_t)256), sms * 8), 256, 0,
                      st>>>(a.pos_q, a.num_q, a.heads, a.pos_dim, gr->dq_pos);
    if ((rc = launched())) return rc;
  }
  if (gr->dk_pos && a.num_k > 0) {
    attn_pos_kernel<<<(unsigned)std::min<int64_t>(ceil_div(a.num_k, (int64_t)256), sms * 8), 256, 0,
                      st>>>(a.pos_k, a.num_k, a.kv_heads, a.pos_dim, gr->dk_pos);
    if ((rc = launched())) return rc;
  }
  if (gr->dsigma) {
    attn_sigma_kernel<<<a.heads, 1024, 0, st>>>(a.pos_q, a.num_q, a.sigma, gr->dsigma);
    if ((rc = launched())) return rc;
  }
  return RA_OK;
}

bool aligned256(const void *p) { return ((uintptr_t)p & 255) == 0; }

}  // namespace

extern "C" {

size_t ra_attn_workspace_bytes(const ra_attn_desc *d, int backward_pass) {
  if (!attn_ok(d)) return 0;
  return std::max<size_t>(256, backward_pass ? bwd_layout(d).total : 0);
}

int ra_attn_forward(const ra_attn_desc *d, const ra_attn_inputs *in, void *out, float *out32,
                    float *stats, void *workspace, size_t workspace_bytes, ra_stream_t stream) {
  if (!attn_ok(d) || !inputs_ok(d, in)) return RA_ERR_INVALID_ARGUMENT;
  if (d->num_q == 0) return RA_OK;
  if (out == nullptr) return RA_ERR_INVALID_ARGUMENT;
  if (workspace == nullptr || !aligned256(workspace) ||
      workspace_bytes < ra_attn_workspace_bytes(d, 0))
    return RA_ERR_WORKSPACE;
  AttnArgs a = args_of(d, in);
  a.out = out, a.out32 = out32, a.stats = (float2 *)stats;
  cudaStream_t st = (cudaStream_t)stream;
  if (d->dtype == RA_F32) return forward<float>(a, st);
  if (d->dtype == RA_BF16) return forward<__nv_bfloat16>(a, st);
  return forward<__half>(a, st);
}

int ra_attn_backward(const ra_attn_desc *d, const ra_attn_inputs *in, const void *dout,
                     const void *out, const float *out32, const float *stats,
                     const ra_attn_grads *grads, void *workspace, size_t workspace_bytes,
                     ra_stream_t stream) {
  if (!attn_ok(d) || !inputs_ok(d, in) || grads == nullptr) return RA_ERR_INVALID_ARGUMENT;
  if (d->num_q > 0 && (dout == nullptr || stats == nullptr || (out == nullptr && out32 == nullptr)))
    return RA_ERR_INVALID_ARGUMENT;
  if (d->pos_dim == 0 && (grads->dq_pos || grads->dk_pos || grads->dsigma))
    return RA_ERR_INVALID_ARGUMENT;
  const AttnBwd b = bwd_layout(d);
  if (workspace == nullptr || !aligned256(workspace) || workspace_bytes < b.total)
    return RA_ERR_WORKSPACE;
  char *ws = (char *)workspace;
  AttnArgs a = args_of(d, in);
  a.out = const_cast<void *>(out), a.out32 = const_cast<float *>(out32);
  a.stats = (float2 *)stats, a.dout = dout, a.delta = (float *)(ws + b.delta);
  a.dq = grads->dq, a.dk = grads->dk, a.dv = grads->dv;
  if (grads->dq_pos || grads->dsigma) a.pos_q = (float4 *)(ws + b.pos_q);
  if (grads->dk_pos) a.pos_k = (float4 *)(ws + b.pos_k);
  cudaStream_t st = (cudaStream_t)stream;
  if (d->dtype == RA_F32) return backward<float>(a, grads, ws, st);
  if (d->dtype == RA_BF16) return backward<__nv_bfloat16>(a, grads, ws, st);
  return backward<__half>(a, grads, ws, st);
}

}  // extern "C"
