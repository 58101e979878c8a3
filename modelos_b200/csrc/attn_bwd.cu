// Windowed attention backward on the 5th-generation tensor cores.
//
//   P = exp(scale q k^T - lse),  dP = dout v^T,  dS = P (dP - delta),
//   delta = sum_d dout out,
//   dq = scale dS k,  dk = scale dS^T q,  dv = P^T dout
//
// Two persistent kernels that add nothing by atomics, so that sums have a fixed order:
// attn_dq walks the key blocks that a tile of 128 query rows sees (3 products
// a block), attn_dkv walks the query blocks, of every query head of
// the group, that see a tile of 128 keys (4 products a block).  One kernel
// with both would need 5 products a block instead of 7, but adds dq in memory
// in an order that changes from run to run.
//
// Both: warps 0-7 element by element (a thread owns a row of TMEM and half of
// the block's columns), warp 8 TMA, warp 9 MMA issuer, another warp zeroes
// rows behind the sequence where they are a product's K dimension, and in
// attn_dkv warp 10 loads lse and delta of the block's queries.  P and dS go
// back into TMEM over S and dP, in the operands' type, as A operands.  While
// the exponentials of one block run, so do the products that use dS of the
// block before.
//
// Measured (16/8 heads of 128, bf16): 8192 tokens, all visible, dq 0.32 ms, dk
// and dv 0.42 ms, delta 0.015: 910 TFLOP/s of the five products that the gradients
// need, 1300 of the seven that run.  8 x 2048 tokens, window 512: 0.14, 0.18 and
// 0.036 ms.
#include <algorithm>

#include "attn_tc.cuh"

namespace pkm {

constexpr int BW_THREADS = 384;
constexpr int BW_REG_ELEM = 216, BW_REG_OTHER = 72;
static_assert(2 * BW_REG_ELEM + BW_REG_OTHER <= 3 * 168, "the block's registers at launch");

template <int DP>
struct BwTile {
  static constexpr int BYTES = AT_T * DP * 2;
  static constexpr int STAGES = 2;
  // two resident tiles, two rings, two output boxes, row statistics
  // (no room is left to round the base up: it has to be aligned)
  static constexpr int SMEM = (2 + 2 * STAGES) * BYTES + 2 * AT_BOX + STAGES * 2 * AT_T * 4 + 256;
  static_assert(SMEM <= 227 * 1024, "shared memory of a block");
};

// P and dS are rounded to the operands' type for their products: the tensor
// cores take two operands of one 16-bit type (attn_exact() has what that costs in
// accuracy and where it is avoided).  In bf16 that is 2^-8 of each
// value, whatever its size.  fp16 has the range 2^-14 to 65504, and neither
// keeps within it: P is 1 / n for n keys seen alike, and |dS| = P |dP - delta| <=
// 2 N, N the norm of a dout row times the largest norm of a v row, is as large or
// small as dout.  So in fp16 both are held times powers of two, taken out again
// when dk, dv and dq are stored: P times 2^14, dS times 2^e with 2^e 2 N <= 2^15
// (and above 2^14), e from the row's own norm in attn_dq and from the largest
// in attn_dkv, where a sum runs over the rows.  What is lost then lies under N 2^-38.
constexpr int BW_P_SHIFT = 14;
template <typename T>
struct Shifted {
  static constexpr bool value = DtOf<T>::value == PKM_DT_F16;
};
__device__ __forceinline__ int ds_shift(float n) {  // e for N = n; 0 without a bound
  return n > 0.f && n < INFINITY ? 13 - ((int)(__float_as_uint(n) >> 23) - 127) : 0;
}
__device__ __forceinline__ float power2(int e) { return __int_as_float((e + 127) << 23); }

// Raises *peak to the square root of the block's largest `square` (none is
// infinite or NaN).  A maximum of non-negative numbers: the order of the updates
// does not show.  One update a block, and only above what was there: an update
// for every row took 30 us for 43000 rows.
__device__ __forceinline__ void raise_peak(float* peak, float old, float square) {
  __shared__ float squares[8];
#pragma unroll
  for (int o = 16; o; o >>= 1) square = fmaxf(square, __shfl_xor_sync(~0u, square, o));
  if ((threadIdx.x & 31) == 0) squares[threadIdx.x >> 5] = square;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 8; ++i) square = fmaxf(square, squares[i]);
    square = sqrtf(square);
    if (square > old) atomicMax(reinterpret_cast<int*>(peak), __float_as_int(square));
  }
}

// ---------------------------------------------------------------------------
// delta = sum over the channels of dout * (out + out_lo): a block takes 128 rows
// of a head, 16 lanes a row, 16 bytes each, four rows in flight a thread.  (From
// out alone, rounded, a row with few visible keys had 1.7 times the rounding error
// of dq, and not 1.4 times.)
// fp16: the norms of dout's rows too, and the largest of dout's and (the first
// v_blocks blocks) of v's rows of each key/value head.
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256)
    attn_delta_kernel(const AttnBwdArgs g, FastDiv by_tiles, FastDiv by_h, FastDiv by_v_tiles, uint32_t v_blocks) {
  const AttnArgs& a = g.f;
  const int d = (threadIdx.x & 15) * 8, rl = threadIdx.x >> 4;
  const bool in = d < a.D;
  constexpr int R = 4;  // rows in flight
  constexpr uint4 zero = {0, 0, 0, 0};
  if (Shifted<T>::value && blockIdx.x < v_blocks) {
    const uint32_t bh = by_v_tiles.div(blockIdx.x);
    const int b = bh / a.Hk, hk = bh % a.Hk, row = (int)(blockIdx.x - bh * by_v_tiles.d) * AT_T + rl;
    const Span sp = attn_span(a.starts, a.ends, b, a.Tk);
    const T* v = static_cast<const T*>(a.v) + b * a.sv.b + hk * a.sv.h + d;
    float* peak = g.peaks + ((int64_t)a.B * a.Hk + bh) * AT_PEAK;
    const float old = __ldcg(peak);
    float largest = 0.f;
#pragma unroll 1
    for (int i = 0; i < AT_T; i += 16 * R) {
      uint4 x[R];
#pragma unroll
      for (int y = 0; y < R; ++y) {
        const int t = row + i + 16 * y;
        x[y] = in && t >= sp.start && t < sp.end ? *reinterpret_cast<const uint4*>(v + t * a.sv.t) : zero;
      }
#pragma unroll
      for (int y = 0; y < R; ++y) {
        float u[8], square = 0.f;
        VecTraits<T>::unpack(x[y], u);
#pragma unroll
        for (int z = 0; z < 8; ++z) square = fmaf(u[z], u[z], square);
#pragma unroll
        for (int o = 8; o; o >>= 1) square += __shfl_xor_sync(~0u, square, o);
        if (square < INFINITY) largest = fmaxf(largest, square);
      }
    }
    raise_peak(peak, old, largest);
    return;
  }
  const uint32_t item = blockIdx.x - v_blocks, bh = by_tiles.div(item), b = by_h.div(bh), h = bh - b * a.Hq;
  const int row = (int)(item - bh * by_tiles.d) * AT_T + rl;
  const T* out = static_cast<const T*>(a.out) + b * a.so.b + h * a.so.h + d;
  const T* out_lo = static_cast<const T*>(a.out_lo) + b * a.so.b + h * a.so.h + d;
  const T* dout = static_cast<const T*>(g.dout) + b * g.sdo.b + h * g.sdo.h + d;
  float* peak = nullptr;
  float old = 0.f, largest = 0.f;
  Span sp{};
  if (Shifted<T>::value) {
    peak = g.peaks + ((int64_t)b * a.Hk + h / a.G) * AT_PEAK;
    old = __ldcg(peak);
    sp = attn_span(a.starts, a.ends, (int)b, a.Tk);
  }
#pragma unroll 1
  for (int i = 0; i < AT_T; i += 16 * R) {
    uint4 x[R], lo[R], y[R];
#pragma unroll
    for (int z = 0; z < R; ++z) {
      const int t = row + i + 16 * z;
      const bool ok = in && t < a.Tq;
      x[z] = ok ? *reinterpret_cast<const uint4*>(out + t * a.so.t) : zero;
      lo[z] = ok ? *reinterpret_cast<const uint4*>(out_lo + t * a.so.t) : zero;
      y[z] = ok ? *reinterpret_cast<const uint4*>(dout + t * g.sdo.t) : zero;
    }
#pragma unroll
    for (int z = 0; z < R; ++z) {
      float u[8], l[8], v[8], sum = 0.f, square = 0.f;
      VecTraits<T>::unpack(x[z], u);
      VecTraits<T>::unpack(lo[z], l);
      VecTraits<T>::unpack(y[z], v);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        sum = fmaf(u[c] + l[c], v[c], sum);
        if (Shifted<T>::value) square = fmaf(v[c], v[c], square);
      }
#pragma unroll
      for (int o = 8; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        if (Shifted<T>::value) square += __shfl_xor_sync(~0u, square, o);
      }
      const int t = row + i + 16 * z;
      if ((threadIdx.x & 15) == 0 && t < a.Tq) g.delta[(int64_t)bh * a.Tq + t] = sum;
      if (Shifted<T>::value && t < a.Tq) {
        if ((threadIdx.x & 15) == 0) g.norms[(int64_t)bh * a.Tq + t] = sqrtf(square);
        const int p = t + a.Tk - a.Tq;
        if (p >= sp.start && p < sp.end && square < INFINITY) largest = fmaxf(largest, square);
      }
    }
  }
  if (Shifted<T>::value) raise_peak(peak, old, largest);
}

// ---------------------------------------------------------------------------
// dq
// ---------------------------------------------------------------------------
// A tile of query rows and the key blocks that it sees.
struct DqItem {
  int b, h, hk, r0, len, start, shift;
  Walk walk;
  int tail;
  __device__ __forceinline__ DqItem(const AttnArgs& a, int item, int tiles) {
    const int heads = a.B * a.Hk, bh = item % heads;
    const int id = tiles - 1 - item / heads;  // late rows first: they see the most keys
    b = bh / a.Hk;
    hk = bh % a.Hk;
    r0 = id / a.G * AT_T;
    h = hk * a.G + id % a.G;
    const Span sp = attn_span(a.starts, a.ends, b, a.Tk);
    start = sp.start;
    len = sp.end - sp.start;
    shift = a.Tk - a.Tq - sp.start;
    int lo, hi;
    at_key_range(r0 + shift, min(r0 + AT_T, a.Tq) - 1 + shift, len, a.window, lo, hi);
    walk = at_key_walk(lo, hi, a.window ? a.sinks : 0);
    tail = walk.count > 0 ? len - walk.block(walk.count - 1) * AT_T : AT_T;
  }
};

// TMEM: S in two buffers (columns 0, 128), dP (256; dS over it: the halves of
// the block's columns at 256 and 320), dq (384).
// EXACT: a second product adds what rounding dS left, which lies behind each half
// of dS.
template <typename T, int DP, bool EXACT>
__global__ void __launch_bounds__(BW_THREADS, 1)
    attn_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo,
                   const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                   const __grid_constant__ CUtensorMap tdq, const AttnBwdArgs g) {
  const AttnArgs& a = g.f;
  using F = BwTile<DP>;
  constexpr int ST = F::STAGES;
  constexpr int FMT = DtOf<T>::value == PKM_DT_BF16 ? 1 : 0;
  extern __shared__ __align__(1024) unsigned char smem[];
  if (smem_u32(smem) & 1023u) {  // swizzled tiles need it (never seen)
    raise_err(a.err, PKM_DEVERR_TIMEOUT);
    return;
  }
  unsigned char* sq = smem;
  unsigned char* sdo = sq + F::BYTES;
  unsigned char* sk = sdo + F::BYTES;
  unsigned char* sv = sk + ST * F::BYTES;
  unsigned char* so = sv + ST * F::BYTES;  // a box of 64 output channels for each half of the threads
  uint64_t* r_full = reinterpret_cast<uint64_t*>(so + 2 * AT_BOX);  // Q and dout
  uint64_t* r_empty = r_full + 1;
  uint64_t* k_full = r_empty + 1;
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* k_tail = v_empty + ST;
  uint64_t* v_tail = k_tail + ST;
  uint64_t* s_full = v_tail + ST;  // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* ds_full = dp_full + 1;
  uint64_t* o_full = ds_full + 1;
  uint64_t* o_empty = o_full + 1;
  uint64_t* drain = o_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (a.Tq + AT_T - 1) / AT_T * a.G;
  Items items(tiles * a.B * a.Hk);
  int item;

  if (threadIdx.x == 0) {
    mbar_init(r_full, 1);
    mbar_init(r_empty, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&k_tail[i], 1);
      mbar_init(&v_tail[i], 1);
    }
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 256);
    mbar_init(o_full, 1);
    mbar_init(o_empty, 256);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  if (warp == 8 && lane == 0) {
    prefetch_tmap(&tq);
    prefetch_tmap(&tdo);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    prefetch_tmap(&tdq);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_dp = tmem + 256, t_dq = tmem + 384;

  if (warp == 8) {
    reg_dec<BW_REG_OTHER>();
    if (lane == 0) {
      uint32_t nr = 0, nb = 0;               // items, blocks
      uint32_t tails = 0, partials = 0;      // a bit a stage: the tail barriers' phase, whether the last copy was partial
      bool ok = true;
      while (ok && items.next(item)) {
        const DqItem w(a, item, tiles);
        if (w.walk.count == 0) continue;
        if (!(ok = at_wait(r_empty, (nr & 1) ^ 1, a.err, abort_flag))) break;
        mbar_arrive_expect_tx(r_full, 2 * F::BYTES);
        for (int x = 0; x < DP / 64; ++x) {
          tma_load_4d(sq + x * AT_BOX, &tq, x * 64, w.r0, w.h, w.b, r_full);
          tma_load_4d(sdo + x * AT_BOX, &tdo, x * 64, w.r0, w.h, w.b, r_full);
        }
        ++nr;
        for (int n = 0; n < w.walk.count; ++n) {
          const int st = nb % ST;
          const uint32_t ph = ((nb / ST) & 1) ^ 1;
          const int row = w.start + w.walk.block(n) * AT_T;
          const bool partial = n == w.walk.count - 1 && w.tail < AT_T;
          uint64_t* kb = partial ? &k_tail[st] : &k_full[st];
          uint64_t* vb = partial ? &v_tail[st] : &v_full[st];
          if (!(ok = at_wait(&k_empty[st], ph, a.err, abort_flag))) break;
          mbar_arrive_expect_tx(kb, F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sk + st * F::BYTES + x * AT_BOX, &tk, x * 64, row, w.hk, w.b, kb);
          if (!(ok = at_wait(&v_empty[st], ph, a.err, abort_flag))) {
            mbar_wait(kb, partial ? (tails >> st) & 1u : (nb / ST) & 1, nullptr);
            break;
          }
          mbar_arrive_expect_tx(vb, F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sv + st * F::BYTES + x * AT_BOX, &tv, x * 64, row, w.hk, w.b, vb);
          partials = (partials & ~(1u << st)) | ((uint32_t)partial << st);
          tails ^= (uint32_t)partial << st;
          ++nb;
        }
      }
      // copies in flight land before the block exits
      if (nr) mbar_wait(r_full, (nr - 1) & 1, nullptr);
      for (uint32_t j = nb > ST ? nb - ST : 0; j < nb; ++j) {
        const uint32_t st = j % ST;
        const bool partial = (partials >> st) & 1u;
        const uint32_t ph = partial ? ((tails >> st) & 1u) ^ 1u : (j / ST) & 1;
        mbar_wait(partial ? &k_tail[st] : &k_full[st], ph, nullptr);
        mbar_wait(partial ? &v_tail[st] : &v_full[st], ph, nullptr);
      }
    }
  } else if (warp == 9) {
    reg_dec<BW_REG_OTHER>();
    {
      constexpr uint32_t ID_S = at_idesc(FMT, AT_T, AT_T, 0, 0);
      constexpr uint32_t ID_O = at_idesc(FMT, AT_T, DP, 0, 1);
      constexpr uint32_t STEP = F::BYTES >> 4;
      const uint32_t q0 = at_desc_k(smem_u32(sq)), d0 = at_desc_k(smem_u32(sdo)), k0 = at_desc_k(smem_u32(sk)),
                     v0 = at_desc_k(smem_u32(sv)), km = at_desc_mn(smem_u32(sk));
      const uint32_t ts = __shfl_sync(~0u, tmem, 0), tp = ts + 256, to = ts + 384;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = at_wait(bar, parity, a.err, abort_flag);
        return (bool)__all_sync(~0u, got);
      };
      uint32_t nb = 0;  // blocks whose dS is done
      auto scores = [&](uint32_t u) {  // S(u) = Q K(u)^T
        const int st = u % ST;
        if (!wait(&k_full[st], (u / ST) & 1)) return false;
        if (elect_one()) {
          at_scores<DP>(ts + (u & 1) * AT_T, q0, k0 + st * STEP, ID_S);
          umma_commit(&s_full[u & 1]);
        }
        __syncwarp();
        return true;
      };
      auto dprobs = [&](uint32_t u, bool last) {  // dP(u) = dout V(u)^T
        const int st = u % ST;
        if (!wait(&v_full[st], (u / ST) & 1)) return false;
        if (elect_one()) {
          at_scores<DP>(tp, d0, v0 + st * STEP, ID_S);
          umma_commit(dp_full);
          umma_commit(&v_empty[st]);
          if (last) umma_commit(r_empty);  // Q and dout are read
        }
        __syncwarp();
        return true;
      };
      uint32_t nr = 0;
      bool ok = true;
      while (ok && items.next(item)) {
        const DqItem w(a, item, tiles);
        if (w.walk.count == 0) continue;
        ok = wait(r_full, nr & 1) && scores(nb) && dprobs(nb, w.walk.count == 1);
        for (int n = 0; n < w.walk.count && ok; ++n, ++nb) {
          const bool more = n + 1 < w.walk.count;
          if (more && !(ok = scores(nb + 1))) break;
          if (n == 0 && !(ok = wait(o_empty, (nr & 1) ^ 1))) break;  // the last item's dq has left TMEM
          if (!(ok = wait(ds_full, nb & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            at_accum<64>(to, tp, km + (nb % ST) * STEP, ID_O, n == 0);  // dq += dS K
            if (EXACT) at_accum<64>(to, tp + 32, km + (nb % ST) * STEP, ID_O, false);
            umma_commit(&k_empty[nb % ST]);
            if (!more) umma_commit(o_full);
          }
          __syncwarp();
          if (more) ok = dprobs(nb + 1, n + 2 == w.walk.count);
        }
        ++nr;
      }
      if (elect_one()) {
        umma_commit(drain);
        mbar_wait(drain, 0, nullptr);
      }
      __syncwarp();
    }
  } else if (warp == 10) {
    reg_dec<BW_REG_OTHER>();
    uint32_t nb = 0, tails = 0;
    while (items.next(item)) {
      const DqItem w(a, item, tiles);
      nb += w.walk.count;
      if (w.walk.count > 0 && w.tail < AT_T) {
        const int st = (nb - 1) % ST;
        const uint32_t ph = (tails >> st) & 1u;
        if (!zero_tail<DP>(sk + st * F::BYTES, w.tail, lane, &k_tail[st], ph, &k_full[st], a.err, abort_flag)) break;
        if (!zero_tail<DP>(sv + st * F::BYTES, w.tail, lane, &v_tail[st], ph, &v_full[st], a.err, abort_flag)) break;
        tails ^= 1u << st;
      }
    }
  } else if (warp == 11) {
    reg_dec<BW_REG_OTHER>();
  } else {
    reg_inc<BW_REG_ELEM>();
    const int half = warp >> 2, rl = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const bool leader = rl == 0;
    const float c = a.scale * AT_LOG2E;
    uint32_t nb = 0, nr = 0;
    bool ok = true;
    while (ok && items.next(item)) {
      const DqItem w(a, item, tiles);
      const Walk walk = w.walk;
      const int row = w.r0 + rl, pr = row + w.shift;
      const bool real = row < a.Tq && pr >= 0 && pr < w.len;
      const int first = w.r0 + w.shift, last = first + AT_T - 1;
      float delta = 0.f, lse = 0.f, f = a.scale;  // f: dq is stored times it
      if (real) {
        const int64_t stat = ((int64_t)w.b * a.Hq + w.h) * a.Tq + row;
        delta = g.delta[stat];
        lse = a.lse[stat] * AT_LOG2E;
        if (Shifted<T>::value) {
          const int e = ds_shift(g.norms[stat] * g.peaks[((int64_t)(a.B + w.b) * a.Hk + w.hk) * AT_PEAK]);
          lse -= e;
          f *= power2(-e);
        }
      }
      for (int n = 0; n < walk.count; ++n, ++nb) {
        ok = at_wait(&s_full[nb & 1], (nb >> 1) & 1, a.err, abort_flag);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        float p[64];
        const uint32_t ts = tmem + lanes + (nb & 1) * AT_T + half * 64;
        tmem_ld_32x32b_x32(ts, reinterpret_cast<uint32_t(&)[32]>(p[0]));
        tmem_ld_32x32b_x32(ts + 32, reinterpret_cast<uint32_t(&)[32]>(p[32]));
        tmem_ld_wait();
#pragma unroll
        for (int x = 0; x < 64; ++x) p[x] = ex2(fmaf(p[x], c, -lse));
        const int j0 = walk.block(n) * AT_T;
        const bool whole = j0 + AT_T - 1 <= first && (a.window == 0 || j0 > last - a.window || j0 + AT_T <= a.sinks);
        if (!whole) {
          const int top = pr - j0, low = a.window ? pr - a.window + 1 - j0 : 0, sink = a.window ? a.sinks - j0 : 0;
#pragma unroll
          for (int x = 0; x < 64; x += 32) {
            const uint32_t see = seen_bits(half * 64 + x, top, low, sink);
#pragma unroll
            for (int y = 0; y < 32; ++y) p[x + y] = see >> y & 1 ? p[x + y] : 0.f;
          }
        }
        ok = at_wait(dp_full, nb & 1, a.err, abort_flag);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        uint32_t d[64], ds[32], lo[EXACT ? 32 : 1];
        tmem_ld_32x32b_x32(t_dp + lanes + half * 64, reinterpret_cast<uint32_t(&)[32]>(d[0]));
        tmem_ld_32x32b_x32(t_dp + lanes + half * 64 + 32, reinterpret_cast<uint32_t(&)[32]>(d[32]));
        tmem_ld_wait();
#pragma unroll
        for (int y = 0; y < 32; ++y) {
          const float x0 = p[2 * y] * (__uint_as_float(d[2 * y]) - delta);
          const float x1 = p[2 * y + 1] * (__uint_as_float(d[2 * y + 1]) - delta);
          ds[y] = pack2<T>(x0, x1);
          if constexpr (EXACT) lo[y] = remainder2<T>(x0, x1, ds[y]);
        }
        tmem_st_32x32b_x32(t_dp + lanes + half * 64, ds);
        if constexpr (EXACT) tmem_st_32x32b_x32(t_dp + lanes + half * 64 + 32, lo);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(ds_full);
      }
      if (walk.count > 0) {
        ok = ok && at_wait(o_full, nr & 1, a.err, abort_flag);
        ++nr;
        tc_fence_after();
      }
      if (!(ok = named_all(1 + half, ok))) break;
      // each half of the threads stores 64 of the channels (the first all of them where there are no more)
      if (DP == 128)
        store_tile<T, 64>(t_dq + lanes + half * 64, so + half * AT_BOX, rl, f, real, walk.count > 0, &tdq, w.r0,
                          w.h, w.b, 1 + half, leader, o_empty, half * 64);
      else if (half == 0)
        store_tile<T, 64>(t_dq + lanes, so, rl, f, real, walk.count > 0, &tdq, w.r0, w.h, w.b, 1, leader,
                          o_empty);
      else if (walk.count > 0)
        mbar_arrive(o_empty);
    }
    if (leader) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// ---------------------------------------------------------------------------
// dk, dv
// ---------------------------------------------------------------------------
// A tile of keys and query blocks that see it, of every head of the group: all
// of them, or (far_tiles) those that the tile's window reaches, or a part of
// those behind, which see its sinks.
struct DkvItem {
  int b, hk, j0, len, start, shift, i_base, i_end, k0, k1, nq, n0, count, tail;
  int slot;   // where partial sums go (-1: dk and dv themselves)
  bool none;  // no tile of keys
  __device__ __forceinline__ DkvItem(const AttnBwdArgs& g, int item) {
    const AttnArgs& a = g.f;
    const int heads = a.B * a.Hk, n_far = heads * g.far_tiles * g.far_parts;
    const bool far = item < n_far;
    if (!far) item -= n_far;
    const int bh = item % heads;
    int r = item / heads;
    b = bh / a.Hk;
    hk = bh % a.Hk;
    const Span sp = attn_span(a.starts, a.ends, b, a.Tk);
    const int off = a.Tk - a.Tq;
    start = sp.start;
    len = sp.end - sp.start;
    i_base = max(0, sp.start - off);  // first query row of the sequence: blocks count from it
    i_end = min(a.Tq, sp.end - off);  // one past the last
    shift = off - sp.start;           // query row -> position
    const int first_tile = start / AT_T;
    const int part = far ? r / g.far_tiles : g.far_parts;
    if (far) r = first_tile + r % g.far_tiles;
    j0 = r * AT_T;  // the first keys are seen by the most queries: they come first
    // positions of the tile's keys, and of the queries that see them
    k0 = j0 - sp.start;
    k1 = min(k0 + AT_T, len) - 1;
    const bool sinks = a.window && k1 >= 0 && k0 < len && max(k0, 0) < a.sinks;
    none = far && !sinks;
    slot = sinks && g.far_tiles ? (bh * g.far_tiles + (r - first_tile)) * (g.far_parts + 1) + part : -1;
    nq = n0 = 0;
    if (k1 >= 0 && k0 < len && !none) {
      const int p_lo = max(max(k0, 0), i_base + shift), p_all = min(len - 1, i_end - 1 + shift);
      const int p_near = a.window ? (int)min((int64_t)p_all, (int64_t)k1 + a.window - 1) : p_all;
      const int p_hi = sinks && !g.far_tiles ? p_all : p_near;
      if (far) {
        // the blocks behind the last one that the window reaches
        const int f0 = ((p_lo <= p_near ? p_near : p_lo) - shift - i_base) / AT_T + (p_lo <= p_near ? 1 : 0);
        const int nf = p_lo <= p_all ? max(0, (p_all - shift - i_base) / AT_T + 1 - f0) : 0;
        n0 = f0 + nf * part / g.far_parts;
        nq = f0 + nf * (part + 1) / g.far_parts - n0;
      } else if (p_lo <= p_hi) {
        n0 = (p_lo - shift - i_base) / AT_T;
        nq = (p_hi - shift - i_base) / AT_T - n0 + 1;
      }
    }
    count = nq * a.G;
    tail = nq > 0 ? i_end - (i_base + (n0 + nq - 1) * AT_T) : AT_T;  // queries in a head's last block
  }
};

// e of attn_dkv, one for a key/value head.
__device__ __forceinline__ int dkv_shift(const AttnBwdArgs& g, int b, int hk) {
  const float* p = g.peaks + ((int64_t)b * g.f.Hk + hk) * AT_PEAK;
  return ds_shift(p[0] * p[(int64_t)g.f.B * g.f.Hk * AT_PEAK]);
}

// Rows of TMEM are keys.  TMEM: S^T (columns 0; P^T over it, the halves of
// the block's queries at 0 and 64), dP^T (128; dS^T over it), dv (256), dk
// (256 + DP).
// FAR: some items are parts, stored in 32 bits (compiled apart: with both ways to
// store in one kernel the compiler spills registers).  EXACT: second products add
// what rounding P and dS left, which lies behind each half of them.
enum DkvMode { DKV_PLAIN, DKV_FAR, DKV_EXACT };
template <typename T, int DP, DkvMode MODE>
__global__ void __launch_bounds__(BW_THREADS, 1)
    attn_dkv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo,
                    const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const __grid_constant__ CUtensorMap tdk, const __grid_constant__ CUtensorMap tdv,
                    const __grid_constant__ CUtensorMap tpk, const __grid_constant__ CUtensorMap tpv,
                    const AttnBwdArgs g) {
  const AttnArgs& a = g.f;
  using F = BwTile<DP>;
  constexpr bool FAR = MODE == DKV_FAR, EXACT = MODE == DKV_EXACT;
  constexpr int ST = F::STAGES;
  constexpr int FMT = DtOf<T>::value == PKM_DT_BF16 ? 1 : 0;
  extern __shared__ __align__(1024) unsigned char smem[];
  if (smem_u32(smem) & 1023u) {  // swizzled tiles need it (never seen)
    raise_err(a.err, PKM_DEVERR_TIMEOUT);
    return;
  }
  unsigned char* sk = smem;
  unsigned char* sv = sk + F::BYTES;
  unsigned char* sq = sv + F::BYTES;
  unsigned char* sdo = sq + ST * F::BYTES;
  unsigned char* so = sdo + ST * F::BYTES;  // a box of 64 channels of dv, one of dk
  float* rows = reinterpret_cast<float*>(so + 2 * AT_BOX);               // [ST][lse, delta][128]
  uint64_t* r_full = reinterpret_cast<uint64_t*>(rows + 2 * AT_T * ST);  // K and V
  uint64_t* r_empty = r_full + 1;
  uint64_t* q_full = r_empty + 1;
  uint64_t* q_empty = q_full + ST;
  uint64_t* o_full_ = q_empty + ST;  // dout
  uint64_t* o_empty = o_full_ + ST;
  uint64_t* l_full = o_empty + ST;  // lse and delta
  uint64_t* l_empty = l_full + ST;
  uint64_t* q_tail = l_empty + ST;  // blocks with rows to be zeroed
  uint64_t* o_tail = q_tail + ST;
  uint64_t* s_full = o_tail + ST;
  uint64_t* dp_full = s_full + 1;
  uint64_t* p_full = dp_full + 1;
  uint64_t* ds_full = p_full + 1;
  uint64_t* done = ds_full + 1;
  uint64_t* acc_empty = done + 1;
  uint64_t* drain = acc_empty + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Items items(((a.Tk + AT_T - 1) / AT_T + g.far_tiles * g.far_parts) * a.B * a.Hk);
  int item;

  if (threadIdx.x == 0) {
    mbar_init(r_full, 1);
    mbar_init(r_empty, 1);
    for (int i = 0; i < ST; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&o_full_[i], 1);
      mbar_init(&o_empty[i], 1);
      mbar_init(&q_tail[i], 1);
      mbar_init(&o_tail[i], 1);
      mbar_init(&l_full[i], 32);
      mbar_init(&l_empty[i], 256);
    }
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(p_full, 256);
    mbar_init(ds_full, 256);
    mbar_init(done, 1);
    mbar_init(acc_empty, 256);
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == 9) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_dp = tmem + 128, t_dv = tmem + 256, t_dk = t_dv + DP;

  if (warp == 8) {
    reg_dec<BW_REG_OTHER>();
    if (lane == 0) {
      uint32_t nr = 0, nb = 0, tails = 0, partials = 0;
      bool ok = true;
      while (ok && items.next(item)) {
        const DkvItem w(g, item);
        if (w.count == 0) continue;
        if (!(ok = at_wait(r_empty, (nr & 1) ^ 1, a.err, abort_flag))) break;
        mbar_arrive_expect_tx(r_full, 2 * F::BYTES);
        for (int x = 0; x < DP / 64; ++x) {
          tma_load_4d(sk + x * AT_BOX, &tk, x * 64, w.j0, w.hk, w.b, r_full);
          tma_load_4d(sv + x * AT_BOX, &tv, x * 64, w.j0, w.hk, w.b, r_full);
        }
        ++nr;
        int h = w.hk * a.G, q = 0;
        for (int n = 0; n < w.count; ++n) {
          const int st = nb % ST;
          const uint32_t ph = ((nb / ST) & 1) ^ 1;
          const int row = w.i_base + (w.n0 + q) * AT_T;
          const bool partial = q == w.nq - 1 && w.tail < AT_T;
          uint64_t* qb = partial ? &q_tail[st] : &q_full[st];
          uint64_t* ob = partial ? &o_tail[st] : &o_full_[st];
          if (!(ok = at_wait(&q_empty[st], ph, a.err, abort_flag))) break;
          mbar_arrive_expect_tx(qb, F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sq + st * F::BYTES + x * AT_BOX, &tq, x * 64, row, h, w.b, qb);
          if (!(ok = at_wait(&o_empty[st], ph, a.err, abort_flag))) {
            mbar_wait(qb, partial ? (tails >> st) & 1u : (nb / ST) & 1, nullptr);
            break;
          }
          mbar_arrive_expect_tx(ob, F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sdo + st * F::BYTES + x * AT_BOX, &tdo, x * 64, row, h, w.b, ob);
          partials = (partials & ~(1u << st)) | ((uint32_t)partial << st);
          tails ^= (uint32_t)partial << st;
          ++nb;
          if (++q == w.nq) {
            q = 0;
            ++h;
          }
        }
      }
      // copies in flight land before the block exits
      if (nr) mbar_wait(r_full, (nr - 1) & 1, nullptr);
      for (uint32_t j = nb > ST ? nb - ST : 0; j < nb; ++j) {
        const uint32_t st = j % ST;
        const bool partial = (partials >> st) & 1u;
        const uint32_t ph = partial ? ((tails >> st) & 1u) ^ 1u : (j / ST) & 1;
        mbar_wait(partial ? &q_tail[st] : &q_full[st], ph, nullptr);
        mbar_wait(partial ? &o_tail[st] : &o_full_[st], ph, nullptr);
      }
    }
  } else if (warp == 9) {
    reg_dec<BW_REG_OTHER>();
    {
      constexpr uint32_t ID_S = at_idesc(FMT, AT_T, AT_T, 0, 0);
      constexpr uint32_t ID_O = at_idesc(FMT, AT_T, DP, 0, 1);
      constexpr uint32_t STEP = F::BYTES >> 4;
      const uint32_t k_ = at_desc_k(smem_u32(sk)), v_ = at_desc_k(smem_u32(sv));
      const uint32_t q_ = at_desc_k(smem_u32(sq)), d_ = at_desc_k(smem_u32(sdo));
      const uint32_t qm = at_desc_mn(smem_u32(sq)), dm = at_desc_mn(smem_u32(sdo));
      const uint32_t us = __shfl_sync(~0u, tmem, 0), up = us + 128, uv = us + 256, uk = uv + DP;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = at_wait(bar, parity, a.err, abort_flag);
        return (bool)__all_sync(~0u, got);
      };
      auto scores = [&](uint32_t u) {  // S^T = K Q(u)^T
        const int st = u % ST;
        if (!wait(&q_full[st], (u / ST) & 1)) return false;
        if (elect_one()) {
          at_scores<DP>(us, k_, q_ + st * STEP, ID_S);
          umma_commit(s_full);
        }
        __syncwarp();
        return true;
      };
      auto dprobs = [&](uint32_t u, bool last) {  // dP^T = V dout(u)^T
        const int st = u % ST;
        if (!wait(&o_full_[st], (u / ST) & 1)) return false;
        if (elect_one()) {
          at_scores<DP>(up, v_, d_ + st * STEP, ID_S);
          umma_commit(dp_full);
          if (last) umma_commit(r_empty);  // K and V are read
        }
        __syncwarp();
        return true;
      };
      uint32_t nr = 0, nb = 0;
      bool ok = true;
      while (ok && items.next(item)) {
        const DkvItem w(g, item);
        if (w.count == 0) continue;
        ok = wait(r_full, nr & 1) && scores(nb) && dprobs(nb, w.count == 1);
        for (int n = 0; n < w.count && ok; ++n, ++nb) {
          const int st = nb % ST;
          const bool more = n + 1 < w.count;
          if (n == 0 && !(ok = wait(acc_empty, (nr & 1) ^ 1))) break;  // the last item's dv, dk have left TMEM
          if (!(ok = wait(p_full, nb & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            at_accum<64>(uv, us, dm + st * STEP, ID_O, n == 0);  // dv += P^T dout
            if (EXACT) at_accum<64>(uv, us + 32, dm + st * STEP, ID_O, false);
            umma_commit(&o_empty[st]);
          }
          __syncwarp();
          if (more && !(ok = scores(nb + 1))) break;
          if (!(ok = wait(ds_full, nb & 1))) break;
          tc_fence_after();
          if (elect_one()) {
            at_accum<64>(uk, up, qm + st * STEP, ID_O, n == 0);  // dk += dS^T Q
            if (EXACT) at_accum<64>(uk, up + 32, qm + st * STEP, ID_O, false);
            umma_commit(&q_empty[st]);
            if (!more) umma_commit(done);
          }
          __syncwarp();
          if (more) ok = dprobs(nb + 1, n + 2 == w.count);
        }
        ++nr;
      }
      if (elect_one()) {
        umma_commit(drain);
        mbar_wait(drain, 0, nullptr);
      }
      __syncwarp();
    }
  } else if (warp == 10) {
    reg_dec<BW_REG_OTHER>();
    uint32_t nb = 0;
    bool ok = true;
    while (ok && items.next(item)) {
      const DkvItem w(g, item);
      // lse less P's shift, delta times what is left of dS's
      constexpr float PS = Shifted<T>::value ? BW_P_SHIFT : 0;
      const float ds = Shifted<T>::value && w.count > 0 ? power2(dkv_shift(g, w.b, w.hk) - BW_P_SHIFT) : 1.f;
      int h = w.hk * a.G, q = 0;
      for (int n = 0; n < w.count; ++n, ++nb) {
        const int st = nb % ST;
        const bool got = at_wait(&l_empty[st], ((nb / ST) & 1) ^ 1, a.err, abort_flag);
        if (!(ok = __all_sync(~0u, got))) break;
        const int row = w.i_base + (w.n0 + q) * AT_T;
        const int64_t base = ((int64_t)w.b * a.Hq + h) * a.Tq;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int r = row + x * 32 + lane;
          const bool in = r < w.i_end;
          rows[(st * 2) * AT_T + x * 32 + lane] = in ? a.lse[base + r] * AT_LOG2E - PS : 0.f;
          rows[(st * 2 + 1) * AT_T + x * 32 + lane] = in ? g.delta[base + r] * ds : 0.f;
        }
        mbar_arrive(&l_full[st]);
        if (++q == w.nq) {
          q = 0;
          ++h;
        }
      }
    }
  } else if (warp == 11) {
    reg_dec<BW_REG_OTHER>();
    // each head of the group ends in the same partial block
    uint32_t nb = 0, ph = 0;  // ph: phase of each stage's tail barriers, a bit a stage
    bool ok = true;
    while (ok && items.next(item)) {
      const DkvItem w(g, item);
      if (w.count > 0 && w.tail < AT_T)
        for (int n = w.nq - 1; n < w.count; n += w.nq) {
          const int st = (nb + n) % ST;
          const uint32_t p = (ph >> st) & 1u;
          if (!(ok = zero_tail<DP>(sq + st * F::BYTES, w.tail, lane, &q_tail[st], p, &q_full[st], a.err, abort_flag)))
            break;
          if (!(ok = zero_tail<DP>(sdo + st * F::BYTES, w.tail, lane, &o_tail[st], p, &o_full_[st], a.err,
                                   abort_flag)))
            break;
          ph ^= 1u << st;
        }
      nb += w.count;
    }
  } else {
    reg_inc<BW_REG_ELEM>();
    const int half = warp >> 2, rl = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + half * 64, td = t_dp + lanes + half * 64;
    const uint32_t rows_s = smem_u32(rows);
    const bool leader = rl == 0;
    const float c = a.scale * AT_LOG2E;
    uint32_t nb = 0, nr = 0;
    bool ok = true;
    while (ok && items.next(item)) {
      const DkvItem w(g, item);
      const int jr = w.j0 + rl - w.start;
      const bool real = w.j0 + rl < a.Tk && jr >= 0 && jr < w.len;
      const int e = Shifted<T>::value && w.count > 0 ? dkv_shift(g, w.b, w.hk) : 0;
      const float ds = power2(e - BW_P_SHIFT);  // (fp16)
      int q = 0;
      for (int n = 0; n < w.count; ++n, ++nb) {
        const int st = nb % ST;
        ok = at_wait(&l_full[st], (nb / ST) & 1, a.err, abort_flag) && at_wait(s_full, nb & 1, a.err, abort_flag);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        const uint32_t lse = rows_s + ((st * 2) * AT_T + half * 64) * 4, delta = lse + AT_T * 4;
        float p[64];
        tmem_ld_32x32b_x32(ts, reinterpret_cast<uint32_t(&)[32]>(p[0]));
        tmem_ld_32x32b_x32(ts + 32, reinterpret_cast<uint32_t(&)[32]>(p[32]));
        tmem_ld_wait();
#pragma unroll
        for (int x = 0; x < 64; x += 4) {
          const float4 e = lds_f4(lse + x * 4);
          p[x] = ex2(fmaf(p[x], c, -e.x));
          p[x + 1] = ex2(fmaf(p[x + 1], c, -e.y));
          p[x + 2] = ex2(fmaf(p[x + 2], c, -e.z));
          p[x + 3] = ex2(fmaf(p[x + 3], c, -e.w));
        }
        const int i0 = w.i_base + (w.n0 + q) * AT_T, q0 = i0 + w.shift;  // the block's first query: row, position
        const bool whole = q0 >= w.k1 && (a.window == 0 || q0 + AT_T - 1 < w.k0 + a.window || w.k1 < a.sinks) &&
                           i0 + AT_T <= w.i_end;
        if (!whole) {
          // columns [low, top) see this row's key
          const int low = jr - q0;
          int top = w.i_end - i0;
          if (a.window && jr >= a.sinks) top = min(top, jr + a.window - q0);
          if (!real) top = 0;
#pragma unroll
          for (int x = 0; x < 64; x += 32) {
            const uint32_t see = seen_bits(half * 64 + x, top - 1, low, 0);
#pragma unroll
            for (int y = 0; y < 32; ++y) p[x + y] = see >> y & 1 ? p[x + y] : 0.f;
          }
        }
        if (++q == w.nq) q = 0;
        uint32_t v[32];
#pragma unroll
        for (int x = 0; x < 32; ++x)
          v[x] = EXACT ? pack2_down<T>(p[2 * x], p[2 * x + 1]) : pack2<T>(p[2 * x], p[2 * x + 1]);
        tmem_st_32x32b_x32(ts, v);
        if constexpr (EXACT) {
          uint32_t first;
#pragma unroll
          for (int x = 0; x < 32; ++x) parts2<T>(p[2 * x], p[2 * x + 1], first, v[x]);
          tmem_st_32x32b_x32(ts + 32, v);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full);
        ok = at_wait(dp_full, nb & 1, a.err, abort_flag);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        uint32_t d[64];
        tmem_ld_32x32b_x32(td, reinterpret_cast<uint32_t(&)[32]>(d[0]));
        tmem_ld_32x32b_x32(td + 32, reinterpret_cast<uint32_t(&)[32]>(d[32]));
        tmem_ld_wait();
#pragma unroll
        for (int y = 0; y < 64; y += 4) {
          const float4 m = lds_f4(delta + y * 4);
          auto diff = [&](uint32_t dp, float m) {
            return Shifted<T>::value ? fmaf(__uint_as_float(dp), ds, -m) : __uint_as_float(dp) - m;
          };
          p[y] *= diff(d[y], m.x);
          p[y + 1] *= diff(d[y + 1], m.y);
          p[y + 2] *= diff(d[y + 2], m.z);
          p[y + 3] *= diff(d[y + 3], m.w);
          v[y / 2] = pack2<T>(p[y], p[y + 1]);
          v[y / 2 + 1] = pack2<T>(p[y + 2], p[y + 3]);
        }
        mbar_arrive(&l_empty[st]);
        tmem_st_32x32b_x32(td, v);
        if constexpr (EXACT) {
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = remainder2<T>(p[2 * x], p[2 * x + 1], v[x]);
          tmem_st_32x32b_x32(td + 32, v);
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(ds_full);
      }
      if (w.count > 0) {
        ok = ok && at_wait(done, nr & 1, a.err, abort_flag);
        ++nr;
        tc_fence_after();
      }
      if (!(ok = named_all(1 + half, ok))) break;
      // the first half of the threads stores dv, the second dk
      const uint32_t acc = (half ? t_dk : t_dv) + lanes;
      const float f = !Shifted<T>::value ? (half ? a.scale : 1.f) : half ? a.scale * power2(-e) : power2(-BW_P_SHIFT);
      if (FAR && w.slot >= 0)
        store_part<DP>(acc, so + half * AT_BOX, rl, f, real, w.count > 0, half ? &tpk : &tpv, a.D, 0, 0, w.slot,
                       1 + half, leader, acc_empty);
      else if (!w.none)
        store_tile<T, DP>(acc, so + half * AT_BOX, rl, f, real, w.count > 0, half ? &tdk : &tdv, w.j0, w.hk, w.b,
                          1 + half, leader, acc_empty);
    }
    if (leader) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

// The parts of the key tiles that hold sinks, summed in their order: 16 lanes a
// row, dk and dv in turn.  Parts are in 32 bits: a part may leave fp16's range
// where the sum does not.
struct FarArgs {
  const float* part[2];  // dk, dv: [slots, 128, D]
};
template <typename T>
__global__ void __launch_bounds__(256) attn_far_join_kernel(const AttnBwdArgs g, const FarArgs f) {
  const AttnArgs& a = g.f;
  const int tile = blockIdx.x / (AT_T / 16), rl = blockIdx.x % (AT_T / 16) * 16 + (threadIdx.x >> 4);
  const int bh = tile / g.far_tiles, ts = tile % g.far_tiles;
  const int b = bh / a.Hk, hk = bh % a.Hk, d = (threadIdx.x & 15) * 8;
  const Span sp = attn_span(a.starts, a.ends, b, a.Tk);
  const int j0 = (sp.start / AT_T + ts) * AT_T, row = j0 + rl, k0 = j0 - sp.start;
  const int len = sp.end - sp.start;
  if (k0 >= len || min(k0 + AT_T, len) <= 0 || max(k0, 0) >= a.sinks || row >= a.Tk || d >= a.D) return;
  const int side = blockIdx.y;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p <= g.far_parts; ++p) {
    float u[8];
    const float4* at = reinterpret_cast<const float4*>(
        f.part[side] + (((int64_t)tile * (g.far_parts + 1) + p) * AT_T + rl) * a.D + d);
    *reinterpret_cast<float4*>(u) = at[0];
    *reinterpret_cast<float4*>(u + 4) = at[1];
#pragma unroll
    for (int y = 0; y < 8; ++y) sum[y] += u[y];
  }
  const Strides3& s = side ? g.sdv : g.sdk;
  *reinterpret_cast<uint4*>(static_cast<T*>(side ? g.dv : g.dk) + b * s.b + hk * s.h + (int64_t)row * s.t + d) =
      make_uint4(pack2<T>(sum[0], sum[1]), pack2<T>(sum[2], sum[3]), pack2<T>(sum[4], sum[5]), pack2<T>(sum[6], sum[7]));
}

// Items for the queries behind a sink's window pay where such a tile's walk
// over all queries is more than half of what a multiprocessor has to do: 1187
// tokens x 3, 12/4 heads: dk and dv 56 -> 40 us; but 2048 x 8, 16/8 heads, where
// it is a third: 183 -> 206.  Many sinks are many such walks, which fill the GPU
// by themselves; and there are only as many parts as make two items a
// multiprocessor.  So the parts' sums take at most 12 * 128 rows of dk and dv for
// each multiprocessor (233 MB for heads of 128), whatever the sizes.
size_t attn_bwd_far(AttnBwdArgs& g) {
  const AttnArgs& a = g.f;
  g.far_tiles = g.far_parts = 0;
  if (!a.window || !a.sinks || !a.Tq || attn_exact(a)) return 0;
  const int64_t heads = (int64_t)a.B * a.Hk, tiles = (a.Tk + AT_T - 1) / AT_T;
  const int64_t all = (a.Tq + AT_T - 1) / AT_T + 1, near = (a.window + AT_T - 1) / AT_T + 2;
  const int64_t walks = (a.sinks - 1) / AT_T + 1, slots = 2 * num_sms();
  if (all < 2 * near || all * slots < heads * (tiles * near + walks * all)) return 0;
  g.far_tiles = (int)walks + 1;  // (they may begin inside a tile)
  g.far_parts = (int)std::min<int64_t>({16, (all - 1) / near, (slots + heads * walks - 1) / (heads * walks)});
  return (size_t)heads * g.far_tiles * (g.far_parts + 1) * AT_T * a.D * 2 * sizeof(float);
}

template <typename T, int DP>
static int attn_bwd_go(const AttnBwdArgs& g, void* partials, cudaStream_t st) {
  const AttnArgs& a = g.f;
  constexpr int dt = DtOf<T>::value;
  constexpr int smem = BwTile<DP>::SMEM;
  // (before the tensor maps: it makes the device's context current on this thread)
  const bool exact = attn_exact(a);
  const auto dq = exact ? attn_dq_kernel<T, DP, true> : attn_dq_kernel<T, DP, false>;
  const auto dkv = g.far_tiles ? attn_dkv_kernel<T, DP, DKV_FAR>
                   : exact     ? attn_dkv_kernel<T, DP, DKV_EXACT>
                               : attn_dkv_kernel<T, DP, DKV_PLAIN>;
  if (cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
      cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_cuda("cudaFuncSetAttribute(attn_bwd)");
  CUtensorMap tq{}, tdo{}, tk, tv, tdq{}, tdk, tdv, tp[2]{};
  int rc;
  if ((rc = attn_tmap(&tk, a.k, dt, a.sk, a.B, a.Hk, a.Tk, a.D)) ||
      (rc = attn_tmap(&tv, a.v, dt, a.sv, a.B, a.Hk, a.Tk, a.D)) ||
      (rc = attn_tmap(&tdk, g.dk, dt, g.sdk, a.B, a.Hk, a.Tk, a.D)) ||
      (rc = attn_tmap(&tdv, g.dv, dt, g.sdv, a.B, a.Hk, a.Tk, a.D)))
    return rc;
  if (a.Tq > 0 && ((rc = attn_tmap(&tq, a.q, dt, a.sq, a.B, a.Hq, a.Tq, a.D)) ||
                   (rc = attn_tmap(&tdo, g.dout, dt, g.sdo, a.B, a.Hq, a.Tq, a.D)) ||
                   (rc = attn_tmap(&tdq, g.dq, dt, g.sdq, a.B, a.Hq, a.Tq, a.D))))
    return rc;
  // partial sums: dk, dv
  const int64_t slots = (int64_t)a.B * a.Hk * g.far_tiles * (g.far_parts + 1);
  FarArgs far{};
  for (int i = 0; i < 2 && slots; ++i) {
    far.part[i] = static_cast<const float*>(partials) + i * slots * AT_T * a.D;
    if ((rc = attn_tmap(&tp[i], far.part[i], PKM_DT_F32, Strides3{(int64_t)AT_T * a.D, 0, a.D}, slots, 1, AT_T, a.D)))
      return rc;
  }
  const int64_t gq = (int64_t)((a.Tq + AT_T - 1) / AT_T) * a.G * a.B * a.Hk;
  const int64_t gk = ((int64_t)((a.Tk + AT_T - 1) / AT_T) + g.far_tiles * g.far_parts) * a.B * a.Hk;
  const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
  if (gq > INT32_MAX / 2 || gk > INT32_MAX / 2 || rows > INT32_MAX - 16)
    return fail(PKM_ERR_UNSUPPORTED, "too many rows");
  const int sms = num_sms();
  if (rows > 0) {
    const int64_t tiles = (a.Tq + AT_T - 1) / AT_T, v_tiles = (a.Tk + AT_T - 1) / AT_T;
    const int64_t v_blocks = Shifted<T>::value ? v_tiles * a.B * a.Hk : 0;
    if (v_blocks &&
        cudaMemsetAsync(g.peaks, 0, (size_t)a.B * a.Hk * 2 * AT_PEAK * sizeof(float), st) != cudaSuccess)
      return check_cuda("cudaMemsetAsync(attn_bwd)");
    attn_delta_kernel<T><<<(unsigned)(tiles * a.B * a.Hq + v_blocks), 256, 0, st>>>(
        g, FastDiv((uint32_t)tiles), FastDiv((uint32_t)a.Hq), FastDiv((uint32_t)v_tiles), (uint32_t)v_blocks);
    dq<<<(unsigned)std::min<int64_t>(gq, sms), BW_THREADS, smem, st>>>(tq, tdo, tk, tv, tdq, g);
  }
  if ((rc = check_cuda("attn_dq"))) return rc;
  dkv<<<(unsigned)std::min<int64_t>(gk, sms), BW_THREADS, smem, st>>>(tq, tdo, tk, tv, tdk, tdv, tp[0], tp[1], g);
  if ((rc = check_cuda("attn_dkv")) || !slots) return rc;
  attn_far_join_kernel<T><<<dim3((unsigned)((int64_t)a.B * a.Hk * g.far_tiles * (AT_T / 16)), 2), 256, 0, st>>>(g, far);
  return check_cuda("attn_far_join");
}

int attn_bwd_launch(const AttnBwdArgs& g, int dtype, void* partials, cudaStream_t st) {
  if (dtype == PKM_DT_BF16)
    return g.f.D > 64 ? attn_bwd_go<__nv_bfloat16, 128>(g, partials, st)
                      : attn_bwd_go<__nv_bfloat16, 64>(g, partials, st);
  return g.f.D > 64 ? attn_bwd_go<__half, 128>(g, partials, st) : attn_bwd_go<__half, 64>(g, partials, st);
}

}  // namespace pkm
