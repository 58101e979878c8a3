// Windowed attention with sink tokens: the entry points and their checks.
#include <algorithm>

#include "attn.cuh"

namespace pkm {

// Sizes and types shared by the entry points; out's layout is checked by them.
static int attn_check(int dtype, int64_t B, int64_t Hq, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D, double scale,
                      int64_t window, int64_t sinks) {
  if (B < 0 || Hq < 0 || Hk < 0 || Tq < 0 || Tk < 0) return fail(PKM_ERR_INVALID_ARG, "negative size");
  if (dtype != PKM_DT_BF16 && dtype != PKM_DT_F16) return fail(PKM_ERR_UNSUPPORTED, "attention takes bf16 or fp16");
  if (D <= 0 || D % 8 || D > 128)
    return fail(PKM_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 128");
  // (without query heads nothing would write dk and dv)
  if (Hk == 0 ? Hq != 0 : Hq == 0 || Hq % Hk != 0)
    return fail(PKM_ERR_INVALID_ARG, "query heads must be a multiple of the key/value heads");
  if (Tk < Tq) return fail(PKM_ERR_INVALID_ARG, "fewer keys than queries");
  if (window < 0 || sinks < 0) return fail(PKM_ERR_INVALID_ARG, "negative window or sinks");
  if (!isfinite(scale)) return fail(PKM_ERR_INVALID_ARG, "scale must be finite");
  if (B > INT32_MAX || Hq > INT32_MAX || B * std::max(Hq, (int64_t)1) > INT32_MAX || Tk > (1 << 29))
    return fail(PKM_ERR_UNSUPPORTED, "more than 2^31 heads or 2^29 rows");
  return PKM_OK;
}

int attn_layout(const void* p, const int64_t* s, int64_t B, int64_t H, int64_t T, const char* what, Strides3* out) {
  if (!p || !s) return fail(PKM_ERR_INVALID_ARG, std::string("null ") + what);
  *out = Strides3{B > 1 ? s[0] : 0, H > 1 ? s[1] : 0, T > 1 ? s[2] : 0};
  if (!aligned16(p) || (out->b | out->h | out->t) & 7 || out->b < 0 || out->h < 0 || out->t < 0 ||
      (B > 1 && !out->b) || (H > 1 && !out->h) || (T > 1 && !out->t))
    return fail(PKM_ERR_INVALID_ARG, std::string(what) + " needs a 16-byte aligned base and positive, aligned strides");
  return PKM_OK;
}

static AttnArgs attn_args(int64_t B, int64_t Hq, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D, double scale,
                          int64_t window, int64_t sinks, const int32_t* starts, const int32_t* ends, uint32_t* err) {
  AttnArgs a{};
  a.B = (int)B;
  a.Hq = (int)Hq;
  a.Hk = (int)Hk;
  a.G = (int)(Hq / Hk);
  a.Tq = (int)Tq;
  a.Tk = (int)Tk;
  a.D = (int)D;
  a.scale = (float)scale;
  // a window or a sink range longer than the rows is the whole row
  a.window = window >= Tk ? 0 : (int)window;
  a.sinks = (int)std::min(sinks, Tk);
  a.splits = 1;
  a.starts = starts;
  a.ends = ends;
  a.err = err;
  return a;
}

}  // namespace pkm

using namespace pkm;

// Partial outputs and sums of a split, in 32 bits.
static size_t attn_fwd_bytes(int64_t B, int64_t Hq, int64_t Tq, int64_t D, int splits) {
  return splits > 1 ? (size_t)splits * B * Hq * Tq * (4 * D + sizeof(float)) : 0;
}

extern "C" int pkm_attn_fwd_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D,
                                      int64_t window, int64_t sinks, size_t* bytes) {
  if (!bytes) return fail(PKM_ERR_INVALID_ARG, "null bytes");
  const int rc = attn_check(PKM_DT_BF16, B, Hq, Hk, Tq, Tk, D, 1.0, window, sinks);
  if (rc) return rc;
  *bytes = 0;
  if (B && Hq && Tq && !attn_few_rows(B, Hk, Hq / Hk, Tq))
    *bytes = attn_fwd_bytes(B, Hq, Tq, D, attn_fwd_splits(B, Hk, Hq / Hk, Tq, Tk, window, sinks));
  return PKM_OK;
}

extern "C" int pkm_attn_fwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, int dtype, int64_t B, int64_t Hq, int64_t Hk,
                            int64_t Tq, int64_t Tk, int64_t D, double scale, int64_t window, int64_t sinks,
                            const int32_t* starts, const int32_t* ends, void* out, const int64_t* out_strides,
                            void* out_lo, float* lse, void* workspace, size_t workspace_bytes,
                            uint32_t* dev_err, void* stream) {
  int rc = attn_check(dtype, B, Hq, Hk, Tq, Tk, D, scale, window, sinks);
  if (rc || B == 0 || Hq == 0 || Tq == 0) return rc;
  AttnArgs a = attn_args(B, Hq, Hk, Tq, Tk, D, scale, window, sinks, starts, ends, dev_err);
  if ((rc = attn_layout(q, q_strides, B, Hq, Tq, "q", &a.sq)) ||
      (rc = attn_layout(k, k_strides, B, Hk, Tk, "k", &a.sk)) ||
      (rc = attn_layout(v, v_strides, B, Hk, Tk, "v", &a.sv)) ||
      (rc = attn_layout(out, out_strides, B, Hq, Tq, "out", &a.so)))
    return rc;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.out_lo = out_lo;
  a.lse = lse;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_lo && !aligned16(out_lo)) return fail(PKM_ERR_INVALID_ARG, "out_lo needs a 16-byte aligned base");
  // Up to 16 query rows to a key/value head: the kernel for few rows, which
  // reads the keys once for all of them (2305 keys, 8 sequences, 2 rows: 12 us,
  // the tiles of 128 rows 54 us).  Its grid has the batch in a dimension of
  // at most 65535.
  if (attn_few_rows(B, Hk, Hq / Hk, Tq)) return attn_decode_launch(a, dtype, st);
  a.splits = attn_fwd_splits(B, Hk, Hq / Hk, Tq, Tk, window, sinks);
  const size_t need = attn_fwd_bytes(B, Hq, Tq, D, a.splits);
  if (need > workspace_bytes || (need && !workspace))
    return fail(PKM_ERR_WORKSPACE, "pkm_attn_fwd: workspace smaller than pkm_attn_fwd_workspace()");
  if (need && !aligned16(workspace)) return fail(PKM_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
  if (a.splits > 1 && B * Hq * Tq > INT32_MAX - 16) return fail(PKM_ERR_UNSUPPORTED, "too many rows");
  return attn_fwd_launch(a, dtype, workspace, st);
}

// delta and the rows' norms, the heads' largest norms, then the partial sums of
// key tiles that hold sinks.
static size_t attn_bwd_rows(int64_t B, int64_t Hq, int64_t Tq) {
  return ((size_t)B * Hq * Tq * sizeof(float) + 255) / 256 * 256;
}
static size_t attn_bwd_stats(int64_t B, int64_t Hq, int64_t Hk, int64_t Tq) {
  return 2 * attn_bwd_rows(B, Hq, Tq) + (size_t)B * Hk * 2 * AT_PEAK * sizeof(float);
}

extern "C" int pkm_attn_bwd_workspace(int64_t B, int64_t Hq, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D,
                                      int64_t window, int64_t sinks, size_t* bytes) {
  if (!bytes) return fail(PKM_ERR_INVALID_ARG, "null bytes");
  const int rc = attn_check(PKM_DT_BF16, B, Hq, Hk, Tq, Tk, D, 1.0, window, sinks);
  if (rc) return rc;
  *bytes = attn_bwd_stats(B, Hq, Hk, Tq);
  if (B && Hq && Tk) {
    AttnBwdArgs g{};
    g.f = attn_args(B, Hq, Hk, Tq, Tk, D, 1.0, window, sinks, nullptr, nullptr, nullptr);
    *bytes += attn_bwd_far(g);
  }
  return PKM_OK;
}

extern "C" int pkm_attn_bwd(const void* q, const int64_t* q_strides, const void* k, const int64_t* k_strides,
                            const void* v, const int64_t* v_strides, const void* out, const int64_t* out_strides,
                            const void* out_lo, const void* dout, const int64_t* dout_strides, const float* lse, int dtype, int64_t B,
                            int64_t Hq, int64_t Hk, int64_t Tq, int64_t Tk, int64_t D, double scale, int64_t window,
                            int64_t sinks, const int32_t* starts, const int32_t* ends, void* dq,
                            const int64_t* dq_strides, void* dk, const int64_t* dk_strides, void* dv,
                            const int64_t* dv_strides, void* workspace, size_t workspace_bytes, uint32_t* dev_err,
                            void* stream) {
  int rc = attn_check(dtype, B, Hq, Hk, Tq, Tk, D, scale, window, sinks);
  if (rc || B == 0 || Hq == 0 || Tk == 0) return rc;
  AttnBwdArgs g{};
  AttnArgs& a = g.f;
  a = attn_args(B, Hq, Hk, Tq, Tk, D, scale, window, sinks, starts, ends, dev_err);
  if ((rc = attn_layout(k, k_strides, B, Hk, Tk, "k", &a.sk)) ||
      (rc = attn_layout(v, v_strides, B, Hk, Tk, "v", &a.sv)) ||
      (rc = attn_layout(dk, dk_strides, B, Hk, Tk, "dk", &g.sdk)) ||
      (rc = attn_layout(dv, dv_strides, B, Hk, Tk, "dv", &g.sdv)))
    return rc;
  if (Tq && ((rc = attn_layout(q, q_strides, B, Hq, Tq, "q", &a.sq)) ||
             (rc = attn_layout(out, out_strides, B, Hq, Tq, "out", &a.so)) ||
             (rc = attn_layout(dout, dout_strides, B, Hq, Tq, "dout", &g.sdo)) ||
             (rc = attn_layout(dq, dq_strides, B, Hq, Tq, "dq", &g.sdq))))
    return rc;
  if (Tq && (!lse || !out_lo || !aligned16(out_lo))) return fail(PKM_ERR_INVALID_ARG, "null lse or out_lo");
  const size_t stats = attn_bwd_stats(B, Hq, Hk, Tq), need = stats + attn_bwd_far(g);
  if (need && !aligned16(workspace)) return fail(PKM_ERR_INVALID_ARG, "workspace must be 16-byte aligned");
  if (workspace_bytes < need || (need && !workspace))
    return fail(PKM_ERR_WORKSPACE, "pkm_attn_bwd: workspace smaller than pkm_attn_bwd_workspace()");
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = const_cast<void*>(out);
  a.out_lo = const_cast<void*>(out_lo);
  a.lse = const_cast<float*>(lse);
  g.dout = dout;
  g.dq = dq;
  g.dk = dk;
  g.dv = dv;
  char* ws = static_cast<char*>(workspace);
  g.delta = reinterpret_cast<float*>(ws);
  g.norms = reinterpret_cast<float*>(ws + attn_bwd_rows(B, Hq, Tq));
  g.peaks = reinterpret_cast<float*>(ws + 2 * attn_bwd_rows(B, Hq, Tq));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return attn_bwd_launch(g, dtype, ws + stats, st);
}
