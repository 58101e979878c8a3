// What the attention kernels share: the call's description, the positions a
// query sees, and the host-side checks.
//
// q [B, Hq, Tq, D], k and v [B, Hk, Tk, D] with element strides for batch,
// head and token (channels contiguous); query head h reads key/value head
// h / (Hq / Hk).  Query i of a sequence stands at row p = i + Tk - Tq; key j
// is visible to it when
//   start <= j < end,  j <= p < end,  p >= start,
//   and  window == 0  or  j > p - window  or  j < start + sinks,
// [start, end) being the sequence's rows ([0, Tk) without the arrays).  A
// query with nothing visible (a row outside) has output 0 and log-sum-exp -inf;
// one that sees a score of NaN or +inf, or only scores of -inf, has output NaN.
#pragma once

#include <math.h>

#include "common.cuh"

namespace pkm {

struct Strides3 {
  int64_t b, h, t;
};

struct AttnArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  void* out_lo;  // what out's rounding left, rounded, in out's layout; may be NULL
  float* lse;    // [B, Hq, Tq], natural log; may be NULL
  Strides3 sq, sk, sv, so;
  int B, Hq, Hk, G, Tq, Tk, D;
  float scale;
  int window, sinks;
  int splits;  // blocks that share an item's keys (1: none)
  const int32_t* starts;  // [B] or NULL
  const int32_t* ends;    // [B] or NULL
  uint32_t* err;
};

constexpr int AT_PEAK = 32;  // a cache line: the updates of different heads do not queue

struct AttnBwdArgs {
  AttnArgs f;
  const void* dout;
  void* dq;
  void* dk;
  void* dv;
  Strides3 sdo, sdq, sdk, sdv;
  float* delta;  // [B, Hq, Tq]: sum over the channels of dout * out
  // fp16 only: the norms of dout's rows [B, Hq, Tq], and for each key/value head
  // the largest of them and of v's rows [2][B, Hk], AT_PEAK numbers apart
  float* norms;
  float* peaks;
  // key tiles that hold sinks are seen by all later queries: those behind the
  // window are items of their own, `far_parts` for each of up to `far_tiles`
  // such tiles of a head (0: no such items), joined afterwards
  int far_tiles, far_parts;
};

// Attention over the 4-bit cache.
struct Kv4Attend {
  const void* q;
  Strides3 sq;
  const uint8_t* codes[2];
  const void* params[2];
  void* out;
  Strides3 so;
  int B, Hq, Hk, G, Tq, cap, D;
  float scale;
  int window, sinks;
  const int32_t* starts;
  const int32_t* lengths;
  uint32_t* err;
};

// Checks a tensor's base and element strides (batch, head, token); the stride
// of a dimension of size 1 becomes 0.
int attn_layout(const void* p, const int64_t* s, int64_t B, int64_t H, int64_t T, const char* what, Strides3* out);

int attn_decode_launch(const AttnArgs& a, int dtype, cudaStream_t st);
int kv4_attend_launch(const Kv4Attend& a, int dtype, cudaStream_t st);
int attn_fwd_launch(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st);
// Whether the kernel for few rows serves a call, and how many blocks share an
// item's keys in the other.
bool attn_few_rows(int64_t B, int64_t Hk, int64_t G, int64_t Tq);
int attn_fwd_splits(int64_t B, int64_t Hk, int64_t G, int64_t Tq, int64_t Tk, int64_t window, int64_t sinks);
// Whether P and dS take part in their products with their rounding's remainders.
bool attn_exact(const AttnArgs& a);
// Sets far_tiles and far_parts; returns the bytes their partial sums take.
size_t attn_bwd_far(AttnBwdArgs& g);
int attn_bwd_launch(const AttnBwdArgs& g, int dtype, void* partials, cudaStream_t st);

// A sequence's rows, clamped into the tensor's.
struct Span {
  int start, end;
};
__device__ __forceinline__ Span attn_span(const int32_t* starts, const int32_t* ends, int b, int rows) {
  Span s;
  s.start = starts ? max(0, min(starts[b], rows)) : 0;
  s.end = ends ? max(s.start, min(ends[b], rows)) : rows;
  return s;
}

}  // namespace pkm
