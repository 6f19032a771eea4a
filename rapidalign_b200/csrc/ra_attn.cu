// ra_attn.cu -- host side of kernel attention (ra_attn.cuh).
#include <algorithm>

#include "ra_attn.cuh"
#include "ra_attn_few.cuh"
#include "ra_attn_few16.cuh"
#include "ra_attn_tc.cuh"
#include "ra_host.h"
#include "ra_tmap.h"

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
  if ((d->test_hooks & ~RA_TEST_NO_MMA) != 0) return false;
  if (d->forward_only != 0 && d->forward_only != 1) return false;
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
  a.qs = {in->q_ptr, (const int4 *)in->q_tiles, d->max_q};
  a.ks = {in->k_ptr, (const int4 *)in->k_tiles, d->max_k};
  a.n_q_tiles = d->q_tiles, a.n_k_tiles = d->k_tiles;
  a.q_pos = d->pos_dim ? in->q_pos : nullptr, a.k_pos = d->pos_dim ? in->k_pos : nullptr;
  a.sigma = in->sigma;
  a.q_mask = in->q_mask, a.k_mask = in->k_mask;
  a.heads = d->heads, a.kv_heads = d->kv_heads, a.dim = d->dim, a.pos_dim = d->pos_dim;
  a.scale = d->scale, a.cap = d->softcap;
  a.status = d->status;
  return a;
}

AttnTcArgs tc_args(const ra_attn_desc *d, const char *state) {
  AttnTcArgs x{};
  x.words = (const unsigned *)state;
  x.no_mma = (d->test_hooks & RA_TEST_NO_MMA) != 0;
  return x;
}

// Head widths the tensor-core kernels take (ra_attn_tc.cuh); other widths and
// 16-bit operands that are not 16-byte aligned go to the warp-per-row kernels.
bool use_tc(const ra_attn_desc *d) { return d->dim <= 128 && d->dim % 8 == 0; }
bool operands_aligned(const ra_attn_desc *d, const ra_attn_inputs *in) {
  if (d->dtype == RA_F32) return true;
  const int64_t s = d->q_row | d->q_head | d->k_row | d->k_head | d->v_row | d->v_head;
  // a stride of 0 (broadcast heads or rows) has no tensor map
  const bool moves = (d->num_q < 2 || d->q_row > 0) && (d->heads < 2 || d->q_head > 0) &&
                     (d->num_k < 2 || (d->k_row > 0 && d->v_row > 0)) &&
                     (d->kv_heads < 2 || (d->k_head > 0 && d->v_head > 0));
  return moves && (s & 7) == 0 &&
         (((uintptr_t)in->q | (uintptr_t)in->k | (uintptr_t)in->v) & 15) == 0;
}

// A few rows a graph: bound by the keys' bytes (ra_attn_few.cuh).
bool use_few(const ra_attn_desc *d) {
  return use_tc(d) && d->max_q * (d->heads / d->kv_heads) <= kFewRows;
}
// The state a backward needs: bounds (fp32 inputs; the backward writes fp16's),
// and the halves of fp32 inputs.
struct AttnState {
  size_t qh, ql, kh, kl, vh, vl, total;
};
size_t words_of(const ra_attn_desc *d, int tensors) {
  return (size_t)tensors * (size_t)d->graphs * (size_t)d->kv_heads;
}
AttnState state_layout(const ra_attn_desc *d) {
  AttnState s{};
  size_t o = 256;
  if (d->forward_only && use_few(d)) {  // reads the inputs as they are
    s.total = o;
    return s;
  }
  if (d->dtype != RA_BF16 && use_tc(d)) o = std::max(o, align256(4 * words_of(d, 4)));
  if (d->dtype == RA_F32 && use_tc(d)) {
    const size_t q = align256(2 * (size_t)d->num_q * d->heads * d->dim);
    const size_t k = align256(2 * (size_t)d->num_k * d->kv_heads * d->dim);
    s.qh = o, s.ql = o + q, o += 2 * q;
    s.kh = o, s.kl = o + k, o += 2 * k;
    s.vh = o, s.vl = o + k, o += 2 * k;
  }
  s.total = o;
  return s;
}

// Key ranges of a row tile: as many as fill the SMs twice, each at least four
// key tiles of the longest graph.
int key_splits(const ra_attn_desc *d, int sms) {
  const int64_t ctas = d->q_tiles * d->heads;
  if (ctas < 1 || ctas >= 2 * sms) return 1;
  int64_t s = 2 * sms / ctas;
  s = std::min<int64_t>(s, ceil_div(d->max_k, (int64_t)64) / 4);
  return s < 1 ? 1 : (int)s;
}

// 16-byte loads of eight columns
bool few_aligned(const ra_attn_desc *d, const ra_attn_inputs *in) {
  const int64_t s = d->q_row | d->q_head | d->k_row | d->k_head | d->v_row | d->v_head;
  return (s & (d->dtype == RA_F32 ? 3 : 7)) == 0 &&
         (((uintptr_t)in->q | (uintptr_t)in->k | (uintptr_t)in->v) & 15) == 0;
}
// Key ranges: as many as fill the SMs once, each at least 512 keys.
int few_splits(const ra_attn_desc *d, int sms) {
  const int64_t ctas = d->graphs * d->kv_heads;
  const int64_t fit = sms * (d->dtype == RA_F32 ? few_ctas(d->max_q * (d->heads / d->kv_heads)) : kFew16Ctas);
  if (ctas < 1 || ctas >= fit) return 1;
  const int64_t s = std::min<int64_t>(fit / ctas, d->max_k / 512);
  return s < 1 ? 1 : (int)s;
}

struct AttnFwd {
  int splits;
  size_t part_o, part_s, total;
};
AttnFwd fwd_layout(const ra_attn_desc *d, int sms) {
  AttnFwd f{};
  f.splits = use_few(d) ? few_splits(d, sms) : use_tc(d) ? key_splits(d, sms) : 1;
  size_t o = 0;
  if (f.splits > 1) {
    const size_t rows = (size_t)f.splits * d->num_q * d->heads;
    f.part_o = o;
    o += align256(4 * rows * d->dim);
    f.part_s = o;
    o += align256(8 * rows);
  }
  f.total = o;
  return f;
}

struct AttnBwd {
  size_t delta, do_top, pos_q, pos_k, gh, gl, total;
};
AttnBwd bwd_layout(const ra_attn_desc *d) {
  AttnBwd b{};
  size_t o = 0;
  b.delta = o;
  o += align256(sizeof(float) * (size_t)d->num_q * d->heads);
  b.do_top = o;
  if (d->dtype != RA_BF16 && use_tc(d)) o += align256(sizeof(float) * (size_t)d->num_q * d->heads);
  b.pos_q = o;
  if (d->pos_dim) o += align256(sizeof(float4) * (size_t)d->num_q * d->heads);
  b.pos_k = o;
  if (d->pos_dim) o += align256(sizeof(float4) * (size_t)d->num_k * d->kv_heads);
  if (d->dtype == RA_F32 && use_tc(d)) {
    const size_t g = align256(2 * (size_t)d->num_q * d->heads * d->dim);
    b.gh = o, b.gl = o + g, o += 2 * g;
  }
  b.total = o;
  return b;
}

unsigned grid_rows(int64_t n, int per) { return (unsigned)ceil_div(n, (int64_t)per); }

AttnPrep prep_of(const AttnArgs &a) {
  AttnPrep p{};
  p.graphs = a.graphs, p.kv_heads = a.kv_heads, p.dim = a.dim;
  return p;
}
int64_t prep_grid(const AttnPrep &p) {
  int64_t tiles = 0;
  for (int t = 0; t < p.count; ++t) tiles = std::max(tiles, p.tiles[t]);
  return tiles * p.kv_heads;
}
template <class T>
int bounds(const AttnPrep &p, unsigned *words, cudaStream_t st) {
  const int64_t n = prep_grid(p);
  if (n > (int64_t)0x7fffffff) return RA_ERR_INVALID_ARGUMENT;
  if (n < 1) return RA_OK;
  attn_bounds_kernel<T><<<dim3((unsigned)n, p.count), kPrepThreads, 0, st>>>(p, words);
  return launched();
}
int halves(const AttnPrep &p, unsigned *words, cudaStream_t st) {
  const int64_t n = prep_grid(p);
  if (n > (int64_t)0x7fffffff) return RA_ERR_INVALID_ARGUMENT;
  if (n < 1) return RA_OK;
  attn_halves_kernel<<<dim3((unsigned)n, p.count), kPrepThreads, 0, st>>>(p, words);
  return launched();
}
// a tensor of the queries' or the keys' rows
void add(AttnPrep &p, const void *x, bool keys, const AttnArgs &a, int64_t row, int64_t head,
         int word, void *hi, void *lo) {
  const int t = p.count++;
  p.x[t] = x, p.row[t] = row, p.head[t] = head;
  p.heads[t] = keys ? a.kv_heads : a.heads;
  p.segs[t] = keys ? a.ks : a.qs, p.tiles[t] = keys ? a.n_k_tiles : a.n_q_tiles;
  p.mask[t] = keys ? a.k_mask : a.q_mask;
  p.word[t] = word, p.hi[t] = (uint16_t *)hi, p.lo[t] = (uint16_t *)lo;
}

// Tensor maps [rows][heads][dim] of an operand, or of its halves.
bool map_heads(CUtensorMap *m, bool bf16, const void *p, int64_t rows, int heads, int dim,
               int64_t row, int64_t head, int cw, int box_rows) {
  std::memset(m, 0, sizeof(*m));
  EncodeTiledFn fn = encode_tiled();
  if (fn == nullptr) return false;
  if (rows < 1) return true;  // no tile is ever loaded
  if (heads < 2) head = dim;  // not used; has to be a valid stride
  if (rows < 2) row = (int64_t)heads * dim;
  const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
  const cuuint64_t strides[2] = {(cuuint64_t)head * 2, (cuuint64_t)row * 2};
  const cuuint32_t box[3] = {(cuuint32_t)cw, 1, (cuuint32_t)box_rows};
  const cuuint32_t es[3] = {1, 1, 1};
  return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
            const_cast<void *>(p), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
            cw == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
int padded_dim(const ra_attn_desc *d) { return d->dim <= 32 ? 32 : d->dim <= 64 ? 64 : 128; }
bool map_operand(const ra_attn_desc *d, AttnMap *m, const void *hi, const void *lo, int64_t rows,
                 int heads, int64_t row, int64_t head, int br) {
  const bool bf16 = d->dtype == RA_BF16;
  const int dp = padded_dim(d), cw = dp == 32 ? 32 : 64;
  return map_heads(&m->hi, bf16, hi, rows, heads, d->dim, row, head, cw, br) &&
         (d->dtype != RA_F32 ||
          map_heads(&m->lo, bf16, lo, rows, heads, d->dim, row, head, cw, br));
}

// What the kernels read: q, k, v as given or the halves in the state, dout
// (`gh`, `gl`; null in the forward).
struct Operands {
  const void *q[2], *k[2], *v[2], *g[2];
  int64_t qr, qh, kr, kh, vr, vh, gr, gh;
};
Operands operands(const ra_attn_desc *d, const ra_attn_inputs *in, char *state, const void *gh,
                  const void *gl) {
  const int64_t qr = (int64_t)d->heads * d->dim, kr = (int64_t)d->kv_heads * d->dim, D = d->dim;
  if (d->dtype != RA_F32)
    return {{in->q, in->q}, {in->k, in->k}, {in->v, in->v}, {gh, gl}, d->q_row, d->q_head,
            d->k_row, d->k_head, d->v_row, d->v_head, qr, D};
  const AttnState s = state_layout(d);
  return {{state + s.qh, state + s.ql}, {state + s.kh, state + s.kl}, {state + s.vh, state + s.vl},
          {gh, gl}, qr, D, kr, D, kr, D, qr, D};
}
// their maps, `br` rows a box
bool map_operands(const ra_attn_desc *d, const Operands &o, int br, AttnTcArgs *x) {
  return map_operand(d, &x->q, o.q[0], o.q[1], d->num_q, d->heads, o.qr, o.qh, br) &&
         map_operand(d, &x->k, o.k[0], o.k[1], d->num_k, d->kv_heads, o.kr, o.kh, br) &&
         map_operand(d, &x->v, o.v[0], o.v[1], d->num_k, d->kv_heads, o.vr, o.vh, br) &&
         (o.g[0] == nullptr ||
          map_operand(d, &x->go, o.g[0], o.g[1], d->num_q, d->heads, o.gr, o.gh, br));
}

template <auto kernel>
int launch(int64_t grid, int threads, int smem, const AttnArgs &a, const AttnTcArgs &x,
           cudaStream_t st) {
  // as much shared memory as there is: the CTAs of an SM hide each other's waits
  static OncePerDevice once;
  if (!once([&] {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
                   cudaSuccess &&
               cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared) == cudaSuccess;
      }))
    return RA_ERR_CUDA;
  if (grid > (int64_t)0x7fffffff) return RA_ERR_INVALID_ARGUMENT;
  if (grid < 1) return RA_OK;
  kernel<<<(unsigned)grid, threads, smem, st>>>(a, x);
  return launched();
}

template <class Kind, int DP>
int tc_forward(const ra_attn_desc *d, const Operands &o, const AttnArgs &a, AttnTcArgs *x,
               cudaStream_t st) {
  using C = FwdCfg<Kind, DP>;
  if (!map_operands(d, o, C::BR, x)) return RA_ERR_INVALID_ARGUMENT;
  return launch<attn_tc_fwd_kernel<Kind, DP>>(a.n_q_tiles * a.heads * x->splits, C::NT, C::smem,
                                              a, *x, st);
}
template <class Kind, int DP>
int tc_backward(const ra_attn_desc *d, const Operands &o, const AttnArgs &a, AttnTcArgs *x,
                cudaStream_t st) {
  using Q = DqCfg<Kind, DP>;
  using K = DkvCfg<Kind, DP>;
  int rc = RA_OK;
  if (!map_operands(d, o, Q::BR, x)) return RA_ERR_INVALID_ARGUMENT;
  if (a.dq || a.pos_q || a.dk)  // dk reads the D that this kernel puts right
    rc = launch<attn_tc_dq_kernel<Kind, DP>>(a.n_q_tiles * a.heads, Q::NT, Q::smem, a, *x, st);
  static_assert(K::BR == Q::BR, "one set of maps");
  if (!rc && (a.dk || a.dv || a.pos_k))
    rc = launch<attn_tc_dkv_kernel<Kind, DP>>(a.n_k_tiles * a.kv_heads, K::NT, K::smem, a, *x, st);
  return rc;
}

template <class T>
int join(const AttnArgs &a, const AttnFwd &f, char *ws, int sms, cudaStream_t st) {
  if (f.splits == 1) return RA_OK;
  const int64_t rows = a.num_q * a.heads;
  if (rows > (int64_t)0x7fffffff) return RA_ERR_INVALID_ARGUMENT;
  float *po = (float *)(ws + f.part_o);
  float2 *ps = (float2 *)(ws + f.part_s);
  // many parts are many loads one after another, which more warps share
  if (f.splits > 32)
    attn_join_many_kernel<T><<<(unsigned)rows, 1024, 0, st>>>(a, f.splits, po, ps);
  else
    attn_join_kernel<T><<<grid_rows(rows, 8), 256, 0, st>>>(a, f.splits, po, ps);
  return launched();
}

int few_launch(void (*kernel)(AttnArgs, int, float *, float2 *), OncePerDevice &once, int smem,
               const AttnArgs &a, const AttnFwd &f, char *ws, cudaStream_t st) {
  if (!once([&] {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) ==
                   cudaSuccess &&
               cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout,
                                    cudaSharedmemCarveoutMaxShared) == cudaSuccess;
      }))
    return RA_ERR_CUDA;
  const int64_t grid = a.graphs * a.kv_heads * f.splits;
  if (grid > (int64_t)0x7fffffff) return RA_ERR_INVALID_ARGUMENT;
  kernel<<<(unsigned)grid, 32 * kFewWarps, smem, st>>>(a, f.splits, (float *)(ws + f.part_o),
                                                       (float2 *)(ws + f.part_s));
  return launched();
}
template <class T, int DP>
int few16(const AttnArgs &a, const AttnFwd &f, char *ws, cudaStream_t st) {
  static OncePerDevice once;
  return few_launch(attn_few16_kernel<T, DP>, once, Few16Cfg<DP>::smem, a, f, ws, st);
}
template <int N, int LPK>
int few32(const AttnArgs &a, const AttnFwd &f, char *ws, cudaStream_t st) {
  static OncePerDevice once;
  return few_launch(attn_few_kernel<N, LPK>, once, few_smem<N>, a, f, ws, st);
}
template <int N>
int few_width(const AttnArgs &a, const AttnFwd &f, char *ws, cudaStream_t st) {
  // a row's scores need lanes of their own: N <= LPK
  return a.dim <= 32   ? few32<N, (N > 4 ? 8 : 4)>(a, f, ws, st)
         : a.dim <= 64 ? few32<N, 8>(a, f, ws, st)
                       : few32<N, 16>(a, f, ws, st);
}
template <class T>
int few_forward(const ra_attn_desc *d, const AttnArgs &a, const AttnFwd &f, char *ws,
                cudaStream_t st) {
  if constexpr (sizeof(T) == 2) {
    return a.dim <= 32   ? few16<T, 32>(a, f, ws, st)
           : a.dim <= 64 ? few16<T, 64>(a, f, ws, st)
                         : few16<T, 128>(a, f, ws, st);
  } else {
    const int64_t rows = d->max_q * (d->heads / d->kv_heads);
    return rows <= 1   ? few_width<1>(a, f, ws, st)
           : rows <= 2 ? few_width<2>(a, f, ws, st)
           : rows <= 4 ? few_width<4>(a, f, ws, st)
                       : few_width<8>(a, f, ws, st);
  }
}

template <class Kind>
int forward(const ra_attn_desc *d, const ra_attn_inputs *in, const AttnArgs &a, char *state,
            char *ws, cudaStream_t st) {
  using T = typename Kind::T;
  if (!use_tc(d) || !operands_aligned(d, in)) {
    attn_row_fwd_kernel<T>
        <<<grid_rows(a.num_q * a.heads, kAttnWarps), 32 * kAttnWarps, 0, st>>>(a);
    return launched();
  }
  const int sms = sm_count();
  const AttnFwd f = fwd_layout(d, sms);
  int rc;
  if (use_few(d) && few_aligned(d, in) && !(Kind::pair && a.neg_m)) {
    rc = few_forward<T>(d, a, f, ws, st);
    return rc ? rc : join<T>(a, f, ws, sms, st);
  }
  AttnTcArgs x = tc_args(d, state);
  if (Kind::pair) {
    const AttnState s = state_layout(d);
    unsigned *words = (unsigned *)state;
    if (cudaMemsetAsync(words, 0, 4 * words_of(d, 3), st) != cudaSuccess) return RA_ERR_CUDA;
    AttnPrep p = prep_of(a);
    add(p, in->q, false, a, d->q_row, d->q_head, kWq, state + s.qh, state + s.ql);
    add(p, in->k, true, a, d->k_row, d->k_head, kWk, state + s.kh, state + s.kl);
    add(p, in->v, true, a, d->v_row, d->v_head, kWv, state + s.vh, state + s.vl);
    if ((rc = bounds<float>(p, words, st))) return rc;
    if ((rc = halves(p, words, st))) return rc;
  }
  x.splits = f.splits;
  x.part_o = (float *)(ws + f.part_o), x.part_s = (float2 *)(ws + f.part_s);
  x.pair_p = a.out32 != nullptr;
  const Operands o = operands(d, in, state, nullptr, nullptr);
  rc = d->dim <= 32   ? tc_forward<Kind, 32>(d, o, a, &x, st)
       : d->dim <= 64 ? tc_forward<Kind, 64>(d, o, a, &x, st)
                      : tc_forward<Kind, 128>(d, o, a, &x, st);
  return rc ? rc : join<T>(a, f, ws, sms, st);
}

template <class Kind>
int backward(const ra_attn_desc *d, const ra_attn_inputs *in, AttnArgs a, const ra_attn_grads *gr,
             char *state, char *ws, cudaStream_t st) {
  using T = typename Kind::T;
  int rc;
  const int sms = sm_count();
  const AttnBwd b = bwd_layout(d);
  const bool tc = use_tc(d) && operands_aligned(d, in);
  if (tc && !Kind::bf16) a.do_top = (float *)(ws + b.do_top);
  if (a.num_q > 0) {
    const float *o32 = Kind::pair ? (const float *)a.out : a.out32;
    if (tc) {
      int lanes = 1;
      while (lanes * 8 < a.dim) lanes <<= 1;
      const unsigned grid = (unsigned)std::min<int64_t>(
          ceil_div(a.num_q * a.heads * lanes, (int64_t)512), (int64_t)sms * 16);
      attn_delta8_kernel<T><<<grid, 256, 0, st>>>((const T *)a.dout, o32, a.num_q, a.heads, a.dim,
                                                  lanes, a.neg_d, a.do_top);
    } else {
      const unsigned grid =
          (unsigned)std::min<int64_t>(ceil_div(a.num_q * a.heads, (int64_t)8), (int64_t)sms * 16);
      attn_delta_kernel<T><<<grid, 256, 0, st>>>((const T *)a.dout, o32, a.num_q, a.heads, a.dim,
                                                 a.neg_d);
    }
    if ((rc = launched())) return rc;
  }
  if (tc) {
    AttnTcArgs x = tc_args(d, state);
    const int64_t qr = (int64_t)d->heads * d->dim;
    const Operands o = operands(d, in, state, Kind::pair ? ws + b.gh : a.dout,
                                Kind::pair ? ws + b.gl : a.dout);
    if (!Kind::bf16) {
      unsigned *words = (unsigned *)state;
      const int first = Kind::pair ? kWdo : kWv;  // kept from the forward: the others
      if (cudaMemsetAsync(words + words_of(d, first), 0, 4 * words_of(d, 4 - first), st) !=
          cudaSuccess)
        return RA_ERR_CUDA;
      AttnPrep p = prep_of(a);
      add(p, a.dout, false, a, qr, d->dim, kWdo, ws + b.gh, ws + b.gl);
      if (!Kind::pair) add(p, in->v, true, a, d->v_row, d->v_head, kWv, nullptr, nullptr);
      if ((rc = bounds<T>(p, words, st))) return rc;
      if (Kind::pair && (rc = halves(p, words, st))) return rc;
    }
    rc = d->dim <= 32   ? tc_backward<Kind, 32>(d, o, a, &x, st)
         : d->dim <= 64 ? tc_backward<Kind, 64>(d, o, a, &x, st)
                        : tc_backward<Kind, 128>(d, o, a, &x, st);
    if (rc) return rc;
  } else {
    if (a.num_q > 0 && (a.dq || a.pos_q)) {
      attn_row_dq_kernel<T>
          <<<grid_rows(a.num_q * a.heads, kAttnWarps), 32 * kAttnWarps, 0, st>>>(a);
      if ((rc = launched())) return rc;
    }
    if (a.num_k > 0 && (a.dk || a.dv || a.pos_k)) {
      attn_row_dkv_kernel<T>
          <<<grid_rows(a.num_k * a.kv_heads, kAttnWarps), 32 * kAttnWarps, 0, st>>>(a);
      if ((rc = launched())) return rc;
    }
  }
  if (gr->dq_pos || gr->dk_pos || gr->dsigma) {
    const AttnPosGrads p{{a.pos_q, a.pos_k},
                         {a.num_q, a.num_k},
                         {a.heads, a.kv_heads},
                         a.pos_dim,
                         {gr->dq_pos, gr->dk_pos},
                         gr->dsigma,
                         a.sigma};
    const int64_t rows = std::max<int64_t>(std::max(a.num_q, a.num_k), 512);
    const dim3 grid((unsigned)std::max<int64_t>(
                        std::min<int64_t>(ceil_div(rows, (int64_t)512), sms * 4),
                        std::min<int64_t>(a.heads, sms)),
                    3);
    attn_pos_kernel<<<grid, 512, 0, st>>>(p);
    if ((rc = launched())) return rc;
  }
  return RA_OK;
}

bool aligned256(const void *p) { return ((uintptr_t)p & 255) == 0; }

}  // namespace

extern "C" {

size_t ra_attn_workspace_bytes(const ra_attn_desc *d, int backward_pass) {
  if (!attn_ok(d)) return 0;
  return std::max<size_t>(256, backward_pass ? bwd_layout(d).total : fwd_layout(d, sm_count()).total);
}

size_t ra_attn_state_bytes(const ra_attn_desc *d) { return attn_ok(d) ? state_layout(d).total : 0; }

int ra_attn_forward(const ra_attn_desc *d, const ra_attn_inputs *in, void *out, float *out32,
                    float *stats, void *state, size_t state_bytes, void *workspace,
                    size_t workspace_bytes, ra_stream_t stream) {
  if (!attn_ok(d) || !inputs_ok(d, in)) return RA_ERR_INVALID_ARGUMENT;
  if (d->num_q == 0) return RA_OK;
  if (d->forward_only &&
      (stats != nullptr || (use_few(d) && d->dtype == RA_F32 && !few_aligned(d, in))))
    return RA_ERR_INVALID_ARGUMENT;
  if (out == nullptr || (((uintptr_t)out | (uintptr_t)out32) & 15)) return RA_ERR_INVALID_ARGUMENT;
  if (workspace == nullptr || !aligned256(workspace) ||
      workspace_bytes < ra_attn_workspace_bytes(d, 0) || state == nullptr || !aligned256(state) ||
      state_bytes < state_layout(d).total)
    return RA_ERR_WORKSPACE;
  AttnArgs a = args_of(d, in);
  a.out = out, a.out32 = out32;
  if (stats) a.neg_m = stats, a.rl = stats + d->num_q * d->heads;
  cudaStream_t st = (cudaStream_t)stream;
  char *sb = (char *)state, *ws = (char *)workspace;
  if (d->dtype == RA_F32) return forward<KindF32>(d, in, a, sb, ws, st);
  if (d->dtype == RA_BF16) return forward<KindBf16>(d, in, a, sb, ws, st);
  return forward<KindF16>(d, in, a, sb, ws, st);
}

int ra_attn_backward(const ra_attn_desc *d, const ra_attn_inputs *in, const void *dout,
                     const void *out, const float *out32, const float *stats,
                     const ra_attn_grads *grads, void *state, size_t state_bytes, void *workspace,
                     size_t workspace_bytes, ra_stream_t stream) {
  if (!attn_ok(d) || !inputs_ok(d, in) || grads == nullptr) return RA_ERR_INVALID_ARGUMENT;
  if (d->forward_only) return RA_ERR_STATE;
  if (d->num_q > 0 && (dout == nullptr || stats == nullptr || (d->dtype == RA_F32 ? out : out32) == nullptr))
    return RA_ERR_INVALID_ARGUMENT;
  if (d->pos_dim == 0 && (grads->dq_pos || grads->dk_pos || grads->dsigma))
    return RA_ERR_INVALID_ARGUMENT;
  const AttnBwd b = bwd_layout(d);
  if (workspace == nullptr || !aligned256(workspace) || workspace_bytes < b.total ||
      state == nullptr || !aligned256(state) || state_bytes < state_layout(d).total)
    return RA_ERR_WORKSPACE;
  if ((((uintptr_t)grads->dq | (uintptr_t)grads->dk | (uintptr_t)grads->dv | (uintptr_t)dout) & 15))
    return RA_ERR_INVALID_ARGUMENT;
  char *sb = (char *)state, *ws = (char *)workspace;
  AttnArgs a = args_of(d, in);
  a.out = const_cast<void *>(out), a.out32 = const_cast<float *>(out32);
  a.neg_m = const_cast<float *>(stats), a.rl = a.neg_m + d->num_q * d->heads;
  a.dout = dout, a.neg_d = (float *)(ws + b.delta);
  a.dq = grads->dq, a.dk = grads->dk, a.dv = grads->dv;
  if (grads->dq_pos || grads->dk_pos || grads->dsigma) a.pos_q = (float4 *)(ws + b.pos_q);
  if (grads->dk_pos) a.pos_k = (float4 *)(ws + b.pos_k);
  cudaStream_t st = (cudaStream_t)stream;
  if (d->dtype == RA_F32) return backward<KindF32>(d, in, a, grads, sb, ws, st);
  if (d->dtype == RA_BF16) return backward<KindBf16>(d, in, a, grads, sb, ws, st);
  return backward<KindF16>(d, in, a, grads, sb, ws, st);
}

}  // extern "C"
