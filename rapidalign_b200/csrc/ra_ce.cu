// ra_ce.cu -- host side of the linear cross entropy (ra_ce.cuh): layout of
// the caller's buffers, choice of tiles, pieces and K slices, launches.
#include <algorithm>

#include "ra_ce.cuh"
#include "ra_ce_few.cuh"
#include "ra_ce_few16.cuh"
#include "ra_host.h"
#include "ra_tmap.h"

namespace {

using namespace ra;

// Rows of a forward launch, and bytes of its partials (8 for each row and 64 or 32
// columns): a table of 131072 takes 8192 rows at a time.
constexpr int64_t kCeRowsPerPass = 32768;
constexpr int64_t kCePartBytes = (int64_t)128 << 20;
constexpr size_t kCePieceBytes = (size_t)512 << 20;  // du of one piece of the vocabulary

bool ce_ok(const ra_ce_desc *d) {
  if (d == nullptr || d->rows < 0 || d->vocab < 1 || d->dim < 1) return false;
  if (d->rows > ((int64_t)1 << 31) - 256 || d->vocab > ((int64_t)1 << 31) - 512 || d->dim > 65536)
    return false;
  if (d->dtype < RA_F32 || d->dtype > RA_F16) return false;
  if (d->ld_x < d->dim || d->ld_w < d->dim) return false;
  if (d->dtype != RA_F32 && ((d->ld_x & 7) || (d->ld_w & 7))) return false;
  if (d->reduction < RA_REDUCE_NONE || d->reduction > RA_REDUCE_MEAN) return false;
  if (!(d->softcap >= 0.f) || !(d->softcap < INFINITY) || !(d->scale - d->scale == 0.f))
    return false;
  if ((d->test_hooks & ~RA_TEST_NO_MMA) != 0) return false;
  if (d->forward_only != 0 && d->forward_only != 1) return false;
  return d->status != nullptr;
}

int pad8(int n) { return (n + 7) & ~7; }

// A few rows: bound by the table's bytes (ra_ce_few.cuh, ra_ce_few16.cuh).  Whole eights of
// columns, and x in shared memory.
bool use_few(const ra_ce_desc *d) {
  return d->rows <= kCeFewRows && d->dim % 8 == 0 &&
         (size_t)d->rows * d->dim * 4 <= kCeFewSmem;
}
// its 16-byte loads of the table
bool few_aligned(const ra_ce_desc *d, const void *w) {
  return d->dtype != RA_F32 || (((uintptr_t)w & 15) == 0 && d->ld_w % 4 == 0);
}

struct CeState {
  size_t stats, xh, xl, wh, wl, total;
};
CeState ce_state(const ra_ce_desc *d) {
  CeState s{};
  size_t o = 256;
  s.stats = o;
  o += align256(sizeof(float2) * (size_t)d->rows);
  // the forward of a few rows reads the inputs as they are
  if (d->dtype == RA_F32 && !(d->forward_only && use_few(d))) {
    const size_t x = align256(2 * (size_t)d->rows * pad8(d->dim));
    const size_t w = align256(2 * (size_t)d->vocab * pad8(d->dim));
    s.xh = o;
    s.xl = o + x;
    s.wh = o + 2 * x;
    s.wl = o + 2 * x + w;
    o += 2 * x + 2 * w;
  }
  s.total = o;
  return s;
}

// Width of the tiles over n columns: 256 unless half of a last tile or of
// the last wave of CTAs would idle; 128 for pairs (TMEM).  One row of tiles
// reads the table once and is bound by its bytes: any better fit counts.
int tile_width(int64_t m_tiles, int64_t n, int sms, bool pairs) {
  if (pairs) return 128;
  auto waves = [&](int tn) {
    const int64_t t = m_tiles * ceil_div(n, (int64_t)tn);
    return (double)(ceil_div(t, (int64_t)sms) * tn);
  };
  return waves(128) < (m_tiles == 1 ? 1.0 : 0.85) * waves(256) ? 128 : 256;
}

// K slices that fill the SMs when there are few tiles, each at least four
// steps long.
int k_slices(int64_t tiles, int64_t steps, int sms) {
  if (tiles < 1 || tiles >= sms) return 1;
  int64_t s = sms / tiles;
  if (s > steps / 4) s = steps / 4;
  return s < 1 ? 1 : (int)s;
}

struct CePlan {
  int sms, elem;
  int64_t mt;             // 128-row tiles of x
  int64_t pass;           // forward: rows of a launch
  int tn_z, parts;
  int few_ctas;
  int64_t piece, ldg;     // vocabulary piece (columns of du)
  int64_t pieces;
  int tn_d;               // tiles over the embedding width
  int sx, sw;             // K slices of dx and dw
  bool direct_x, direct_w;
  size_t f_part, f_zt, f_blocks, f_total;
  size_t b_coef, b_unit, b_xh, b_xl, b_hi, b_lo, b_px, b_pw, b_total;
};

CePlan ce_plan(const ra_ce_desc *d, int sms) {
  CePlan p{};
  p.sms = sms;
  const bool split = d->dtype == RA_F32;
  p.elem = split ? 4 : 2;
  p.mt = ceil_div(d->rows, (int64_t)kGmM);
  p.tn_z = tile_width(ceil_div(std::min<int64_t>(d->rows, kCeRowsPerPass), (int64_t)kGmM), d->vocab,
                      sms, split);
  p.parts = kGmParts * (int)ceil_div(d->vocab, (int64_t)p.tn_z);
  p.pass = kCePartBytes / ((int64_t)sizeof(float2) * p.parts) / kGmM * kGmM;
  p.pass = std::min<int64_t>(std::max<int64_t>(p.pass, kGmM), kCeRowsPerPass);
  const int64_t pass = std::min<int64_t>(d->rows, p.pass);
  const int few_rows = kCeFewWarps * (split ? 2 : kCeFew16Rows);  // a CTA, at least
  p.few_ctas = (int)std::min<int64_t>(ceil_div(d->vocab, (int64_t)few_rows), split ? 2 * sms : sms);
  size_t o = 0;
  p.f_part = o;
  o += align256(sizeof(float2) * (size_t)p.parts * (size_t)(ceil_div(pass, (int64_t)kGmM) * kGmM));
  o += align256(sizeof(float2) * (size_t)p.few_ctas * kCeFewRows);
  p.f_zt = o;
  o += align256(sizeof(float) * (size_t)d->rows);
  p.f_blocks = o;
  o += align256(sizeof(double2) * (size_t)ceil_div(d->rows, (int64_t)8));
  p.f_total = o;

  const int64_t rows_pad = p.mt * kGmM;
  int64_t piece = (int64_t)(kCePieceBytes / ((size_t)p.elem * (size_t)std::max<int64_t>(rows_pad, 1)));
  piece = std::max<int64_t>(256, piece / 256 * 256);
  const int64_t all = ceil_div(d->vocab, (int64_t)256) * 256;
  p.pieces = ceil_div(all, piece);
  p.piece = ceil_div(ceil_div(all, p.pieces), (int64_t)256) * 256;  // even pieces
  p.pieces = ceil_div(d->vocab, p.piece);
  p.ldg = p.piece;
  p.tn_d = d->dim <= 128 ? 128 : tile_width(p.mt, d->dim, sms, split);
  const int64_t nt = ceil_div((int64_t)d->dim, (int64_t)p.tn_d);
  p.sx = k_slices(p.mt * nt, ceil_div(std::min<int64_t>(p.piece, d->vocab), (int64_t)kGmK), sms);
  p.sw = k_slices(ceil_div(std::min<int64_t>(p.piece, d->vocab), (int64_t)kGmM) * nt,
                  ceil_div(d->rows, (int64_t)kGmK), sms);
  p.direct_x = p.sx == 1 && p.pieces == 1;
  p.direct_w = p.sw == 1;
  o = 0;
  p.b_coef = o;
  o += align256(sizeof(float2) * (size_t)d->rows);
  p.b_unit = o;  // rows in units: the units, and x in them
  if (d->dtype != RA_BF16) {
    o += align256(sizeof(float) * (size_t)d->rows);
    const size_t x = align256(2 * (size_t)d->rows * pad8(d->dim));
    p.b_xh = o;
    o += x;
    p.b_xl = o;
    if (split) o += x;
  }
  const size_t g = align256(2 * (size_t)rows_pad * (size_t)p.ldg);
  p.b_hi = o;
  o += g;
  p.b_lo = o;
  if (split) o += g;
  p.b_px = o;
  if (!p.direct_x) o += align256(sizeof(float) * (size_t)p.sx * (size_t)d->rows * d->dim);
  p.b_pw = o;
  if (!p.direct_w) o += align256(sizeof(float) * (size_t)p.sw * (size_t)p.piece * d->dim);
  p.b_total = o;
  return p;
}

template <int TN, bool BF16, GmOp OP, bool A_MN, bool B_MN, class Epi>
int launch_gemm(const GmMaps &maps, const GmShape &s, const Epi &epi, int sms, cudaStream_t st) {
  const size_t smem = kGmSmem;
  auto k = gemm16_kernel<TN, BF16, OP, A_MN, B_MN, Epi>;
  static OncePerDevice once;
  if (!once([&] {
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) ==
               cudaSuccess;
      }))
    return RA_ERR_CUDA;
  const int64_t units = (int64_t)s.m_tiles * s.n_tiles * s.slices;
  if (units < 1 || units > (int64_t)0x7ff00000) return RA_ERR_INVALID_ARGUMENT;
  k<<<(unsigned)std::min<int64_t>(units, sms), kGmThreads, smem, st>>>(maps, s, epi);
  return launched();
}

template <bool BF16, bool PAIRS, bool A_MN, bool B_MN, class Epi>
int launch_gemm(int tn, const GmMaps &maps, const GmShape &s, const Epi &epi, int sms,
                cudaStream_t st) {
  if constexpr (PAIRS) {
    // a gradient's K is long; the logits' is often one round
    if constexpr (!A_MN && !B_MN)
      if (s.k_steps <= kGmRound)
        return launch_gemm<128, BF16, kGmPairs1, A_MN, B_MN>(maps, s, epi, sms, st);
    return launch_gemm<128, BF16, kGmPairs, A_MN, B_MN>(maps, s, epi, sms, st);
  } else {
    return tn == 256 ? launch_gemm<256, BF16, kGmOne, A_MN, B_MN>(maps, s, epi, sms, st)
                     : launch_gemm<128, BF16, kGmOne, A_MN, B_MN>(maps, s, epi, sms, st);
  }
}

struct Operands {  // 16-bit x and w, or their halves
  const uint16_t *xh, *xl, *wh, *wl;
  int64_t ldx, ldw;
};
Operands operands(const ra_ce_desc *d, const void *x, const void *w, char *state) {
  if (d->dtype != RA_F32)
    return {(const uint16_t *)x, (const uint16_t *)x, (const uint16_t *)w, (const uint16_t *)w,
            d->ld_x, d->ld_w};
  const CeState s = ce_state(d);
  const int ld = pad8(d->dim);
  return {(const uint16_t *)(state + s.xh), (const uint16_t *)(state + s.xl),
          (const uint16_t *)(state + s.wh), (const uint16_t *)(state + s.wl), ld, ld};
}

unsigned grid_for(int64_t n, int sms) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(n, (int64_t)256), (int64_t)sms * 8));
}

bool aligned(const void *p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// logits of x rows [r0, r0 + rows) against w rows [v0, v0 + cols)
bool logit_maps(GmMaps *m, bool bf16, const Operands &op, int dim, int64_t r0, int64_t rows,
                int64_t v0, int64_t cols, int tn) {
  return map16(&m->a_hi, bf16, op.xh + r0 * op.ldx, rows, dim, op.ldx, kGmM) &&
         map16(&m->a_lo, bf16, op.xl + r0 * op.ldx, rows, dim, op.ldx, kGmM) &&
         map16(&m->b_hi, bf16, op.wh + v0 * op.ldw, cols, dim, op.ldw, tn) &&
         map16(&m->b_lo, bf16, op.wl + v0 * op.ldw, cols, dim, op.ldw, tn);
}

template <bool PAIRS>
CeLogit<PAIRS> logit_of(const ra_ce_desc *d, const CeHead *head) {
  return {d->scale, d->softcap, head};
}

GmShape shape_of(const ra_ce_desc *d, const CePlan &p, int64_t mt, int64_t nt, int64_t k, int slices,
                 int m_fast) {
  const bool no_mma = (d->test_hooks & RA_TEST_NO_MMA) != 0;
  return {(int)mt, (int)nt, (int)ceil_div(k, (int64_t)kGmK), slices, m_fast,
          no_mma ? 4096u : kTcSpinLimit, no_mma, d->status};
}

// fp32 inputs as pairs of halves, in the state
int halves(const ra_ce_desc *d, const CePlan &p, const void *x, const void *w, char *sb,
           cudaStream_t st) {
  const CeState sl = ce_state(d);
  CeHead *head = (CeHead *)sb;
  const CeMatrix<float> mx{(const float *)x, d->rows, d->ld_x, d->dim, nullptr, &head->amax_x,
                           (__half *)(sb + sl.xh), (__half *)(sb + sl.xl)};
  const CeMatrix<float> mw{(const float *)w, d->vocab, d->ld_w, d->dim, nullptr, &head->amax_w,
                           (__half *)(sb + sl.wh), (__half *)(sb + sl.wl)};
  const dim3 grid(grid_for(std::max(d->rows, d->vocab) * (pad8(d->dim) / 8), p.sms), 2);
  ce_amax_kernel<<<grid, 256, 0, st>>>(mx, mw);
  int rc = launched();
  if (rc) return rc;
  ce_split_kernel<<<grid, 256, 0, st>>>(mx, mw);
  return launched();
}

// x in its rows' units, in the workspace: what dw multiplies
template <class T>
int rows_in_units(const ra_ce_desc *d, const CePlan &p, const void *x, CeHead *head, char *ws,
                  cudaStream_t st) {
  if (cudaMemsetAsync(&head->amax_xu, 0, 4, st) != cudaSuccess) return RA_ERR_CUDA;
  const CeMatrix<T> m{(const T *)x, d->rows, d->ld_x, d->dim, (const float *)(ws + p.b_unit),
                      &head->amax_xu, (__half *)(ws + p.b_xh),
                      sizeof(T) == 4 ? (__half *)(ws + p.b_xl) : nullptr};
  const unsigned grid = grid_for(d->rows * (pad8(d->dim) / 8), p.sms);
  ce_amax_kernel<T><<<grid, 256, 0, st>>>(m, m);
  int rc = launched();
  if (rc) return rc;
  ce_split_kernel<T><<<grid, 256, 0, st>>>(m, m);
  return launched();
}

template <int N, int LPK>
int few32(const ra_ce_desc *d, const CePlan &p, const float *x, const float *w,
          const int64_t *target, char *ws, cudaStream_t st) {
  auto k = ce_few_kernel<N, LPK>;
  static OncePerDevice once;
  if (!once([&] {
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    (int)kCeFewSmem) == cudaSuccess;
      }))
    return RA_ERR_CUDA;
  k<<<(unsigned)p.few_ctas, 32 * kCeFewWarps, (size_t)d->rows * d->dim * 4, st>>>(
      x, d->ld_x, w, d->ld_w, (int)d->rows, d->vocab, d->dim, d->scale, d->softcap, target,
      (float2 *)(ws + p.f_part), (float *)(ws + p.f_zt));
  return launched();
}
template <int N>
int few_width(const ra_ce_desc *d, const CePlan &p, const float *x, const float *w,
              const int64_t *target, char *ws, cudaStream_t st) {
  return d->dim <= 64    ? few32<N, 8>(d, p, x, w, target, ws, st)
         : d->dim <= 128 ? few32<N, 16>(d, p, x, w, target, ws, st)
                         : few32<N, 32>(d, p, x, w, target, ws, st);
}
template <class T>
int few16(const ra_ce_desc *d, const CePlan &p, const T *x, const T *w, const int64_t *target,
          char *ws, cudaStream_t st) {
  auto k = ce_few16_kernel<T>;
  static OncePerDevice once;
  if (!once([&] {
        return cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                    kCeFew16MostSmem) == cudaSuccess;
      }))
    return RA_ERR_CUDA;
  k<<<(unsigned)p.few_ctas, 32 * kCeFewWarps, ce_few16_smem((int)d->rows, d->dim), st>>>(
      x, d->ld_x, w, d->ld_w, (int)d->rows, d->vocab, d->dim, d->scale, d->softcap, target,
      (float2 *)(ws + p.f_part), (float *)(ws + p.f_zt));
  return launched();
}
int few_forward(const ra_ce_desc *d, const CePlan &p, const void *xv, const void *wv,
                const int64_t *target, char *ws, cudaStream_t st) {
  if (d->dtype == RA_BF16)
    return few16(d, p, (const __nv_bfloat16 *)xv, (const __nv_bfloat16 *)wv, target, ws, st);
  if (d->dtype == RA_F16)
    return few16(d, p, (const __half *)xv, (const __half *)wv, target, ws, st);
  const float *x = (const float *)xv, *w = (const float *)wv;
  return d->rows <= 1   ? few_width<1>(d, p, x, w, target, ws, st)
         : d->rows <= 2 ? few_width<2>(d, p, x, w, target, ws, st)
         : d->rows <= 4 ? few_width<4>(d, p, x, w, target, ws, st)
                        : few_width<8>(d, p, x, w, target, ws, st);
}

// The rows' losses from their parts.  Many rows: 8 threads a row in CTAs of 256
// (65537 rows of 132 parts: 29 us, with 32 threads a row 65 us); few: all of
// 1024 threads on 8 rows.
int join_rows(const ra_ce_desc *d, const float2 *part, int64_t ld, int parts, int64_t r0,
              int64_t rows, const int64_t *target, float *loss, float *lse, char *sb, char *ws,
              const CePlan &p, cudaStream_t st) {
  const CeState sl = ce_state(d);
  CeHead *head = (CeHead *)sb;
  const float *zt = (const float *)(ws + p.f_zt);
  float2 *stats = (float2 *)(sb + sl.stats);
  double2 *blocks = (double2 *)(ws + p.f_blocks);
  if (d->rows <= 8)
    ce_rows_kernel<8, 128><<<1, 1024, 0, st>>>(part, ld, parts, r0, rows, d->rows, d->vocab, target,
                                               d->ignore_index, zt, d->reduction, loss, lse, stats,
                                               head, blocks);
  else if (d->rows <= 4096)
    ce_rows_kernel<32, 32><<<(unsigned)ceil_div(rows, (int64_t)32), 1024, 0, st>>>(
        part, ld, parts, r0, rows, d->rows, d->vocab, target, d->ignore_index, zt, d->reduction,
        loss, lse, stats, head, blocks);
  else
    ce_rows_kernel<32, 8><<<(unsigned)ceil_div(rows, (int64_t)32), 256, 0, st>>>(
        part, ld, parts, r0, rows, d->rows, d->vocab, target, d->ignore_index, zt, d->reduction,
        loss, lse, stats, head, blocks);
  return launched();
}

template <class T, bool BF16, bool SPLIT>
int backward(const ra_ce_desc *d, const CePlan &p, const Operands &op, bool units,
             const int64_t *target, T *dx, T *dw, char *state, char *ws, cudaStream_t st) {
  const CeState sl = ce_state(d);
  CeHead *head = (CeHead *)state;
  uint16_t *gh = (uint16_t *)(ws + p.b_hi), *gl = (uint16_t *)(ws + (SPLIT ? p.b_lo : p.b_hi));
  float *px = (float *)(ws + p.b_px), *pw = (float *)(ws + p.b_pw);
  const int dim = d->dim;
  const int64_t nt = ceil_div((int64_t)dim, (int64_t)p.tn_d);
  const float undo = d->scale / kCeGradScale<BF16>;
  const CeAlpha al_x{undo, &head->amax_g, SPLIT ? &head->amax_w : nullptr};
  const CeAlpha al_w{undo, &head->amax_g,
                     units ? &head->amax_xu : SPLIT ? &head->amax_x : nullptr};
  const float *unit = units ? (const float *)(ws + p.b_unit) : nullptr;
  // x as dw multiplies it
  const uint16_t *xh = units ? (const uint16_t *)(ws + p.b_xh) : op.xh;
  const uint16_t *xl = !units ? op.xl : SPLIT ? (const uint16_t *)(ws + p.b_xl) : xh;
  const int64_t ldx = units ? pad8(dim) : op.ldx;
  for (int64_t i = 0; i < p.pieces; ++i) {
    const int64_t v0 = i * p.piece, cols = std::min<int64_t>(p.piece, d->vocab - v0);
    GmMaps m;
    const int tn = tile_width(p.mt, cols, p.sms, SPLIT);
    if (!logit_maps(&m, BF16, op, dim, 0, d->rows, v0, cols, tn)) return RA_ERR_INVALID_ARGUMENT;
    CeEpiGrad<BF16, SPLIT> eg{logit_of<SPLIT>(d, head), d->rows, d->vocab, v0, target,
                              (const float2 *)(state + sl.stats), (const float2 *)(ws + p.b_coef),
                              head, gh, gl, p.ldg};
    int rc;
    const GmShape sz = shape_of(d, p, p.mt, ceil_div(cols, (int64_t)tn), dim, 1, 1);
    rc = launch_gemm<BF16, SPLIT, false, false>(tn, m, sz, eg, p.sms, st);
    if (rc) return rc;
    if (dx != nullptr) {
      if (!map16(&m.a_hi, BF16, gh, d->rows, cols, p.ldg, kGmM) ||
          !map16(&m.a_lo, BF16, gl, d->rows, cols, p.ldg, kGmM) ||
          !map16(&m.b_hi, BF16, op.wh + v0 * op.ldw, cols, dim, op.ldw, kGmK) ||
          !map16(&m.b_lo, BF16, op.wl + v0 * op.ldw, cols, dim, op.ldw, kGmK))
        return RA_ERR_INVALID_ARGUMENT;
      const int slices = std::min<int>(p.sx, (int)ceil_div(cols, (int64_t)kGmK));
      CeEpiOut<T> eo{al_x, d->rows, dim, p.direct_x ? dx : nullptr, px, i > 0, unit};
      const GmShape s = shape_of(d, p, p.mt, nt, cols, slices, 0);
      rc = launch_gemm<BF16, SPLIT, false, true>(p.tn_d, m, s, eo, p.sms, st);
      if (rc) return rc;
    }
    if (dw != nullptr) {
      if (!map16(&m.a_hi, BF16, gh, d->rows, cols, p.ldg, kGmK) ||
          !map16(&m.a_lo, BF16, gl, d->rows, cols, p.ldg, kGmK) ||
          !map16(&m.b_hi, BF16, xh, d->rows, dim, ldx, kGmK) ||
          !map16(&m.b_lo, BF16, xl, d->rows, dim, ldx, kGmK))
        return RA_ERR_INVALID_ARGUMENT;
      CeEpiOut<T> eo{al_w, cols, dim, p.direct_w ? dw + v0 * dim : nullptr, pw, 0, nullptr};
      const GmShape s = shape_of(d, p, ceil_div(cols, (int64_t)kGmM), nt, d->rows, p.sw, 0);
      rc = launch_gemm<BF16, SPLIT, true, true>(p.tn_d, m, s, eo, p.sms, st);
      if (rc) return rc;
      if (!p.direct_w) {
        ce_join_kernel<T><<<grid_for(cols * dim, p.sms), 256, 0, st>>>(pw, p.sw, cols * dim, al_w,
                                                                       dw + v0 * dim);
        if ((rc = launched())) return rc;
      }
    }
  }
  if (dx != nullptr && !p.direct_x) {
    ce_join_kernel<T><<<grid_for(d->rows * dim, p.sms), 256, 0, st>>>(px, p.sx, d->rows * dim, al_x,
                                                                      dx);
    return launched();
  }
  return RA_OK;
}

}  // namespace

extern "C" {

size_t ra_ce_state_bytes(const ra_ce_desc *d) { return ce_ok(d) ? ce_state(d).total : 0; }

size_t ra_ce_workspace_bytes(const ra_ce_desc *d, int backward_pass) {
  if (!ce_ok(d)) return 0;
  const CePlan p = ce_plan(d, sm_count());
  return std::max<size_t>(256, backward_pass ? p.b_total : p.f_total);
}

int ra_ce_forward(const ra_ce_desc *d, const void *x, const void *w, const int64_t *target,
                  float *loss, float *lse, void *state, size_t state_bytes, void *workspace,
                  size_t workspace_bytes, ra_stream_t stream) {
  if (!ce_ok(d) || w == nullptr) return RA_ERR_INVALID_ARGUMENT;
  if (loss == nullptr && (d->rows > 0 || d->reduction != RA_REDUCE_NONE))
    return RA_ERR_INVALID_ARGUMENT;
  if (d->rows > 0 && (x == nullptr || target == nullptr || lse == nullptr))
    return RA_ERR_INVALID_ARGUMENT;
  if (d->dtype != RA_F32 && (!aligned(x, 16) || !aligned(w, 16))) return RA_ERR_INVALID_ARGUMENT;
  cudaStream_t st = (cudaStream_t)stream;
  const CeState sl = ce_state(d);
  const CePlan p = ce_plan(d, sm_count());
  if (state == nullptr || state_bytes < sl.total || !aligned(state, 256) || workspace == nullptr ||
      workspace_bytes < p.f_total || !aligned(workspace, 256))
    return RA_ERR_WORKSPACE;
  char *sb = (char *)state, *ws = (char *)workspace;
  CeHead *head = (CeHead *)sb;
  if (cudaMemsetAsync(head, 0, 256, st) != cudaSuccess) return RA_ERR_CUDA;
  int rc;
  if (d->rows == 0) {  // the mean of no losses is NaN (all bits set), their sum 0
    if (d->reduction == RA_REDUCE_NONE) return RA_OK;
    return cudaMemsetAsync(loss, d->reduction == RA_REDUCE_MEAN ? 0xff : 0, 4, st) == cudaSuccess
               ? RA_OK
               : RA_ERR_CUDA;
  }
  const bool few = use_few(d) && few_aligned(d, w);
  if (d->forward_only && use_few(d) && !few) return RA_ERR_INVALID_ARGUMENT;
  if (few) {
    if ((rc = few_forward(d, p, x, w, target, ws, st))) return rc;
    return join_rows(d, (const float2 *)(ws + p.f_part), kCeFewRows, p.few_ctas, 0, d->rows, target,
                     loss, lse, sb, ws, p, st);
  }
  if (d->dtype == RA_F32 && (rc = halves(d, p, x, w, sb, st))) return rc;
  const bool bf16 = d->dtype == RA_BF16;
  const Operands op = operands(d, x, w, sb);
  float2 *part = (float2 *)(ws + p.f_part);
  float *zt = (float *)(ws + p.f_zt);
  for (int64_t r0 = 0; r0 < d->rows; r0 += p.pass) {
    const int64_t rows = std::min<int64_t>(p.pass, d->rows - r0);
    const int64_t mt = ceil_div(rows, (int64_t)kGmM);
    GmMaps m;
    if (!logit_maps(&m, bf16, op, d->dim, r0, rows, 0, d->vocab, p.tn_z))
      return RA_ERR_INVALID_ARGUMENT;
    const GmShape s =
        shape_of(d, p, mt, ceil_div(d->vocab, (int64_t)p.tn_z), d->dim, 1, 1);
    if (d->dtype == RA_F32) {
      const CeEpiLse<true> e{logit_of<true>(d, head), rows, d->vocab, target + r0, part, mt * kGmM,
                             zt + r0};
      rc = launch_gemm<false, true, false, false>(p.tn_z, m, s, e, p.sms, st);
    } else {
      const CeEpiLse<false> e{logit_of<false>(d, head), rows, d->vocab, target + r0, part,
                              mt * kGmM, zt + r0};
      rc = bf16 ? launch_gemm<true, false, false, false>(p.tn_z, m, s, e, p.sms, st)
                : launch_gemm<false, false, false, false>(p.tn_z, m, s, e, p.sms, st);
    }
    if (rc) return rc;
    rc = join_rows(d, part, mt * kGmM, p.parts, r0, rows, target, loss, lse, sb, ws, p, st);
    if (rc) return rc;
  }
  return RA_OK;
}

int ra_ce_backward(const ra_ce_desc *d, const void *x, const void *w, const int64_t *target,
                   const float *g_loss, const float *g_lse, void *dx, void *dw, void *state,
                   size_t state_bytes, void *workspace, size_t workspace_bytes,
                   ra_stream_t stream) {
  if (!ce_ok(d) || w == nullptr) return RA_ERR_INVALID_ARGUMENT;
  if (d->forward_only) return RA_ERR_STATE;
  if (d->rows > 0 && (x == nullptr || target == nullptr)) return RA_ERR_INVALID_ARGUMENT;
  if (d->dtype != RA_F32 && (!aligned(x, 16) || !aligned(w, 16))) return RA_ERR_INVALID_ARGUMENT;
  if (!aligned(dx, 16) || !aligned(dw, 16)) return RA_ERR_INVALID_ARGUMENT;
  if (dx == nullptr && dw == nullptr) return RA_OK;
  cudaStream_t st = (cudaStream_t)stream;
  const CeState sl = ce_state(d);
  const CePlan p = ce_plan(d, sm_count());
  if (state == nullptr || state_bytes < sl.total || !aligned(state, 256) || workspace == nullptr ||
      workspace_bytes < p.b_total || !aligned(workspace, 256))
    return RA_ERR_WORKSPACE;
  char *sb = (char *)state, *ws = (char *)workspace;
  CeHead *head = (CeHead *)sb;
  const size_t es = d->dtype == RA_F32 ? 4 : 2;
  if (d->rows == 0) {
    if (dw != nullptr &&
        cudaMemsetAsync(dw, 0, es * (size_t)d->vocab * d->dim, st) != cudaSuccess)
      return RA_ERR_CUDA;
    return RA_OK;
  }
  // Coefficients of rows that may lie apart: fp16 holds each row in its own unit.
  // (Those of a sum or mean of the losses are all alike; bf16 has the range.)
  const bool units = d->dtype != RA_BF16 && (d->reduction == RA_REDUCE_NONE || g_lse != nullptr);
  if (cudaMemsetAsync(&head->amax_g, 0, 4, st) != cudaSuccess) return RA_ERR_CUDA;
  ce_coef_kernel<<<grid_for(d->rows, p.sms), 256, 0, st>>>(
      target, d->rows, d->vocab, d->ignore_index, d->reduction, g_loss, g_lse, head,
      (float2 *)(ws + p.b_coef), units ? (float *)(ws + p.b_unit) : nullptr);
  int rc;
  if ((rc = launched())) return rc;
  if (units && dw != nullptr) {
    rc = d->dtype == RA_F32 ? rows_in_units<float>(d, p, x, head, ws, st)
                            : rows_in_units<__half>(d, p, x, head, ws, st);
    if (rc) return rc;
  }
  // The forward of a few rows made no halves if w lay aligned then; where it
  // lies now says nothing about that.
  if (d->dtype == RA_F32 && use_few(d) && (rc = halves(d, p, x, w, sb, st))) return rc;
  const Operands op = operands(d, x, w, sb);
  if (d->dtype == RA_F32)
    return backward<float, false, true>(d, p, op, units, target, (float *)dx, (float *)dw, sb, ws,
                                        st);
  if (d->dtype == RA_BF16)
    return backward<__nv_bfloat16, true, false>(d, p, op, units, target, (__nv_bfloat16 *)dx,
                                                (__nv_bfloat16 *)dw, sb, ws, st);
  return backward<__half, false, false>(d, p, op, units, target, (__half *)dx, (__half *)dw, sb, ws,
                                        st);
}

}  // extern "C"
