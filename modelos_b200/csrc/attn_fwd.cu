// Windowed attention forward on the 5th-generation tensor cores.
//
// One persistent CTA to a multiprocessor takes items of two tiles of 128 query
// rows that share a key/value head (two query heads at the same rows when
// heads are grouped) and walks the blocks of 128 keys that either sees, one
// pass with a running maximum and sum.  The next item's copies and first
// products run while the last one's output is stored.
//   warps 0-3, 4-7  softmax of tile 0, 1: a thread owns a row; it reads its
//                   128 scores from TMEM, writes the probabilities back over
//                   them in the operands' type (the tensor cores take two
//                   operands of one 16-bit type; attn_exact() has what that
//                   costs in accuracy and where it is avoided), and keeps
//                   maximum and sum in registers;
//   warp 8          TMA: the two Q tiles once, K and V blocks into two-stage
//                   rings;
//   warp 9          MMA issuer: S_i = Q_i K^T (both from shared memory) and
//                   O_i += P_i V (P_i from TMEM);
//   warp 10         zeroes the rows of a V block that lie behind the sequence;
//   warp 11         completes the third warpgroup, whose registers go to the
//                   softmax (a row's 128 scores stay in registers).
// TMEM: S_0, S_1 (128 columns each; P_i over the first half of S_i) and O_0,
// O_1.  The products of one tile run while the other tile's softmax does.
// O is rescaled only when a row's maximum has grown by more than 2^8 over the
// one in use: a probability is then at most 2^8, exact in the accumulator, and
// the common factor cancels in the final division.  The softmax warps rescale
// it themselves: S_i(n)'s arrival says that O_i's last product is done.
//
// Measured (16/8 heads of 128, bf16): 8192 tokens, all visible, 0.25 ms (1080
// TFLOP/s of visible work); 16384 tokens, window 2048 and 64 sinks, 0.28 ms (940).
// In the first of these an iteration takes 3900 cycles where its 32 products need
// 2048 (469000 cycles, 119 iterations in the busiest block, 112 in the average
// one; tensor pipe 50%, issue slots 37%): the chain scores - softmax - product of
// one tile, of which the other tile's hides a half.  Neither fewer
// special-function exponentials nor an earlier hand-over of half of P shortened it.
#include <algorithm>
#include <cstring>

#include "attn_tc.cuh"

namespace pkm {

// Three warpgroups: 168 registers a thread at launch, of which the third
// (copies, products) hands all but 72 to the softmax: 2 * 216 + 72 = 3 * 168.
constexpr int FW_THREADS = 384;
constexpr int FW_REG_SOFTMAX = 216, FW_REG_OTHER = 72;
static_assert(2 * FW_REG_SOFTMAX + FW_REG_OTHER <= 3 * 168, "the block's registers at launch");

template <int DP>
struct FwTile {
  static constexpr int BYTES = AT_T * DP * 2;  // a Q, K or V tile
  static constexpr int STAGES = 2;
  static constexpr int SMEM = (2 + 2 * STAGES) * BYTES + 2 * AT_BOX + 1024 + 256;
};

// Two query tiles of one key/value head and the key blocks that either sees.
struct FwItem {
  int b, hk, pair, nt, len, start, shift;  // shift: query row -> position in the sequence
  Walk walk;
  int count;  // blocks of this item's part of the walk
  int tail;   // the sequence's rows in the last one
  int ob;     // batch of the output: the partial outputs of a split lie behind one another
  __device__ __forceinline__ int block(int n) const { return walk.block(n); }
  __device__ __forceinline__ FwItem(const AttnArgs& a, int item, int tiles) {
    int part = 0;
    if (a.splits > 1) {
      part = item % a.splits;
      item /= a.splits;
    }
    const int heads = a.B * a.Hk, bh = item % heads;
    pair = (tiles + 1) / 2 - 1 - item / heads;  // late rows, which see the most keys, first
    b = bh / a.Hk;
    hk = bh % a.Hk;
    const Span sp = attn_span(a.starts, a.ends, b, a.Tk);
    start = sp.start;
    len = sp.end - sp.start;
    shift = a.Tk - a.Tq - sp.start;
    nt = min(2, tiles - 2 * pair);
    int lo = INT32_MAX, hi = 0;
    for (int i = 0; i < nt; ++i) {
      const int r0 = (2 * pair + i) / a.G * AT_T;
      int l, h;
      at_key_range(r0 + shift, min(r0 + AT_T, a.Tq) - 1 + shift, len, a.window, l, h);
      lo = min(lo, l);
      hi = max(hi, h);
    }
    walk = at_key_walk(lo, hi, a.window ? a.sinks : 0);
    count = walk.count;
    if (a.splits > 1) {
      // (the sinks' blocks all go to the first part)
      const int c0 = part ? max(walk.count * part / a.splits, walk.head) : 0;
      const int c1 = max(walk.count * (part + 1) / a.splits, walk.head);
      if (part) {
        walk.from += c0 - walk.head;
        walk.head = 0;
      }
      count = c1 - c0;
    }
    tail = count > 0 ? len - block(count - 1) * AT_T : AT_T;
    ob = part * a.B + b;
  }
};

// PART: items are parts of a split, stored in 32 bits (compiled apart: with both
// ways to store in one kernel the compiler spills registers).  EXACT: a second
// product adds what rounding the probabilities left; they lie behind P, over the
// second half of S_i.
enum FwMode { FW_PLAIN, FW_PART, FW_EXACT };
template <typename T, int DP, FwMode MODE>
__global__ void __launch_bounds__(FW_THREADS, 1)
    attn_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                    const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tout,
                    const __grid_constant__ CUtensorMap tlo, const AttnArgs a) {
  using F = FwTile<DP>;
  constexpr bool PART = MODE == FW_PART, EXACT = MODE == FW_EXACT;
  constexpr int ST = F::STAGES;
  constexpr int FMT = DtOf<T>::value == PKM_DT_BF16 ? 1 : 0;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  unsigned char* sq = smem;
  unsigned char* sk = sq + 2 * F::BYTES;
  unsigned char* sv = sk + ST * F::BYTES;
  unsigned char* so = sv + ST * F::BYTES;  // a box of 64 output channels for each tile
  uint64_t* bars = reinterpret_cast<uint64_t*>(so + 2 * AT_BOX);
  uint64_t* q_full = bars;            // [2]
  uint64_t* q_empty = q_full + 2;     // [2]
  uint64_t* k_full = q_empty + 2;     // [ST]
  uint64_t* k_empty = k_full + ST;    // [ST]
  uint64_t* v_full = k_empty + ST;    // [ST]
  uint64_t* v_empty = v_full + ST;    // [ST]
  uint64_t* s_full = v_empty + ST;    // [2]
  uint64_t* p_full = s_full + 2;      // [2]
  uint64_t* o_full = p_full + 2;      // [2]
  uint64_t* o_empty = o_full + 2;     // [2]
  uint64_t* v_tail = o_empty + 2;     // [ST]
  uint64_t* drain = v_tail + ST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (a.Tq + AT_T - 1) / AT_T * a.G;
  Items items((tiles + 1) / 2 * a.B * a.Hk * a.splits);
  int item;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], AT_T);
      mbar_init(&o_full[i], 1);
      mbar_init(&o_empty[i], AT_T);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_tail[i], 1);
    }
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
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
    prefetch_tmap(&tout);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 256;

  // Every role walks the same items; the counters below number a barrier's
  // uses over all of them.
  if (warp == 8) {
    reg_dec<FW_REG_OTHER>();
    if (lane == 0) {
      uint32_t nq0 = 0, nq1 = 0, nk = 0, nv = 0;
      uint32_t tails = 0, partials = 0;  // a bit a stage: v_tail's phase, whether its last copy was partial
      bool ok = true;
      while (ok && items.next(item)) {
        const FwItem w(a, item, tiles);
        if (w.count == 0) continue;
        for (int i = 0; i < w.nt && ok; ++i) {
          const int id = 2 * w.pair + i;
          if (!(ok = at_wait(&q_empty[i], ((i ? nq1 : nq0) & 1) ^ 1, a.err, abort_flag))) break;
          mbar_arrive_expect_tx(&q_full[i], F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sq + i * F::BYTES + x * AT_BOX, &tq, x * 64, id / a.G * AT_T, w.hk * a.G + id % a.G, w.b,
                        &q_full[i]);
          (i ? nq1 : nq0)++;
        }
        for (int n = 0; n < w.count && ok; ++n) {
          const int row = w.start + w.block(n) * AT_T;
          int st = nk % ST;
          if (!(ok = at_wait(&k_empty[st], ((nk / ST) & 1) ^ 1, a.err, abort_flag))) break;
          mbar_arrive_expect_tx(&k_full[st], F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sk + st * F::BYTES + x * AT_BOX, &tk, x * 64, row, w.hk, w.b, &k_full[st]);
          ++nk;
          st = nv % ST;
          if (!(ok = at_wait(&v_empty[st], ((nv / ST) & 1) ^ 1, a.err, abort_flag))) break;
          const bool partial = n == w.count - 1 && w.tail < AT_T;
          uint64_t* vb = partial ? &v_tail[st] : &v_full[st];
          partials = (partials & ~(1u << st)) | ((uint32_t)partial << st);
          tails ^= (uint32_t)partial << st;
          mbar_arrive_expect_tx(vb, F::BYTES);
          for (int x = 0; x < DP / 64; ++x)
            tma_load_4d(sv + st * F::BYTES + x * AT_BOX, &tv, x * 64, row, w.hk, w.b, vb);
          ++nv;
        }
      }
      // copies in flight land before the block exits
      if (nq0) mbar_wait(&q_full[0], (nq0 - 1) & 1, nullptr);
      if (nq1) mbar_wait(&q_full[1], (nq1 - 1) & 1, nullptr);
      for (uint32_t j = nk > ST ? nk - ST : 0; j < nk; ++j) mbar_wait(&k_full[j % ST], (j / ST) & 1, nullptr);
      for (uint32_t j = nv > ST ? nv - ST : 0; j < nv; ++j) {
        const uint32_t st = j % ST;
        if ((partials >> st) & 1u)
          mbar_wait(&v_tail[st], ((tails >> st) & 1u) ^ 1u, nullptr);
        else
          mbar_wait(&v_full[st], (j / ST) & 1, nullptr);
      }
    }
  } else if (warp == 9) {
    reg_dec<FW_REG_OTHER>();
    {
      constexpr uint32_t ID_S = at_idesc(FMT, AT_T, AT_T, 0, 0);
      constexpr uint32_t ID_O = at_idesc(FMT, AT_T, DP, 0, 1);
      constexpr uint32_t STEP = F::BYTES >> 4;  // a tile, in the descriptors' units
      const uint32_t q0 = at_desc_k(smem_u32(sq)), k0 = at_desc_k(smem_u32(sk)), v0 = at_desc_mn(smem_u32(sv));
      const uint32_t ts = __shfl_sync(~0u, tmem, 0), to = ts + 256;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        const bool got = at_wait(bar, parity, a.err, abort_flag);
        return (bool)__all_sync(~0u, got);
      };
      uint32_t nq0 = 0, nq1 = 0, nk = 0, nv = 0, np0 = 0, np1 = 0;  // items of a tile, blocks of K, V, P
      bool ok = true;
      while (ok && items.next(item)) {
        const FwItem w(a, item, tiles);
        if (w.count == 0) continue;
        ok = wait(&k_full[nk % ST], (nk / ST) & 1);
        for (int i = 0; i < w.nt && ok; ++i) {
          ok = wait(&q_full[i], (i ? nq1 : nq0) & 1);
          if (ok && elect_one()) {  // S_i = Q_i K(0)^T
            at_scores<DP>(ts + i * AT_T, q0 + i * STEP, k0 + (nk % ST) * STEP, ID_S);
            umma_commit(&s_full[i]);
            if (i == w.nt - 1) umma_commit(&k_empty[nk % ST]);
            if (w.count == 1) umma_commit(&q_empty[i]);
          }
          __syncwarp();
        }
        ++nk;
        for (int n = 0; n < w.count && ok; ++n) {
          const int st = nv % ST, nx = nk % ST;
          const bool more = n + 1 < w.count;
          ok = wait(&v_full[st], (nv / ST) & 1);
          if (more) ok = ok && wait(&k_full[nx], (nk / ST) & 1);
          for (int i = 0; i < w.nt && ok; ++i) {
            // the last item's output has left O_i
            if (n == 0 && !(ok = wait(&o_empty[i], ((i ? nq1 : nq0) & 1) ^ 1))) break;
            if (!(ok = wait(&p_full[i], (i ? np1 : np0) & 1))) break;
            if (i)
              ++np1;
            else
              ++np0;
            tc_fence_after();
            if (elect_one()) {
              at_accum<32>(to + i * DP, ts + i * AT_T, v0 + st * STEP, ID_O, n == 0);  // O_i += P_i V(n)
              if (EXACT) at_accum<32>(to + i * DP, ts + i * AT_T + 64, v0 + st * STEP, ID_O, false);
              if (i == w.nt - 1) umma_commit(&v_empty[st]);
              if (more) {  // S_i = Q_i K(n + 1)^T
                at_scores<DP>(ts + i * AT_T, q0 + i * STEP, k0 + nx * STEP, ID_S);
                umma_commit(&s_full[i]);
                if (i == w.nt - 1) umma_commit(&k_empty[nx]);
                if (n + 2 == w.count) umma_commit(&q_empty[i]);
              } else {
                umma_commit(&o_full[i]);
              }
            }
            __syncwarp();
          }
          ++nv;
          if (more) ++nk;
        }
        ++nq0;
        if (w.nt > 1) ++nq1;
      }
      if (elect_one()) {
        umma_commit(drain);  // every product completes before TMEM is released
        mbar_wait(drain, 0, nullptr);
      }
      __syncwarp();
    }
  } else if (warp == 10) {
    reg_dec<FW_REG_OTHER>();
    // a probability of 0 does not silence a NaN in V
    uint32_t nv = 0, tails = 0;
    while (items.next(item)) {
      const FwItem w(a, item, tiles);
      nv += w.count;
      if (w.count > 0 && w.tail < AT_T) {
        const int st = (nv - 1) % ST;
        if (!zero_tail<DP>(sv + st * F::BYTES, w.tail, lane, &v_tail[st], (tails >> st) & 1u, &v_full[st], a.err,
                           abort_flag))
          break;
        tails ^= 1u << st;
      }
    }
  } else if (warp == 11) {
    reg_dec<FW_REG_OTHER>();
  } else {
    reg_inc<FW_REG_SOFTMAX>();
    const int i = warp >> 2;
    const int rl = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t ts = tmem + lanes + i * AT_T;
    const uint32_t to = tmem_o + lanes + i * DP;
    const bool leader = rl == 0;
    // scores in powers of two (at scale 0 a hidden score must still give 0);
    // a hidden score becomes `hidden`, which times c is -inf
    const float c = copysignf(fmaxf(fabsf(a.scale) * AT_LOG2E, 1e-37f), a.scale);
    const uint32_t hidden = c < 0.f ? 0x7f800000u : 0xff800000u;
    uint32_t ns = 0, no = 0;  // blocks, items
    bool ok = true;
    while (ok && items.next(item)) {
      const FwItem w(a, item, tiles);
      if (i >= w.nt) continue;
      const int first = (2 * w.pair + i) / a.G * AT_T + w.shift;  // positions of the tile's rows
      const int last = first + AT_T - 1, pr = first + rl;
      float m = -INFINITY, l = 0.f;
      for (int n = 0; n < w.count; ++n, ++ns) {
        ok = at_wait(&s_full[i], ns & 1, a.err, abort_flag);
        if (!(ok = __all_sync(~0u, ok))) break;
        tc_fence_after();
        const int j0 = w.block(n) * AT_T;
        // some row of the tile does not see some key of the block
        const bool whole = j0 + AT_T - 1 <= first && (a.window == 0 || j0 > last - a.window || j0 + AT_T <= a.sinks);
        const int top = pr - j0;                                 // last visible column
        const int low = a.window ? pr - a.window + 1 - j0 : 0;   // first column of the window
        const int sink = a.window ? a.sinks - j0 : 0;            // columns before it are sinks
        uint32_t s[AT_T];
#pragma unroll
        for (int x = 0; x < 4; ++x) tmem_ld_32x32b_x32(ts + x * 32, reinterpret_cast<uint32_t(&)[32]>(s[x * 32]));
        tmem_ld_wait();
        if (!whole) {
#pragma unroll
          for (int x = 0; x < AT_T; x += 32) {
            const uint32_t see = seen_bits(x, top, low, sink);
#pragma unroll
            for (int y = 0; y < 32; ++y) s[x + y] = see >> y & 1 ? s[x + y] : hidden;
          }
        }
        float mx;
        {
          float m4[4];
          if (c < 0.f) {
#pragma unroll
            for (int y = 0; y < 4; ++y) m4[y] = fminf(__uint_as_float(s[y]), __uint_as_float(s[4 + y]));
#pragma unroll
            for (int x = 8; x < AT_T; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                m4[y] = fminf(fminf(m4[y], __uint_as_float(s[x + y])), __uint_as_float(s[x + 4 + y]));
            mx = fminf(fminf(m4[0], m4[1]), fminf(m4[2], m4[3]));
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) m4[y] = fmaxf(__uint_as_float(s[y]), __uint_as_float(s[4 + y]));
#pragma unroll
            for (int x = 8; x < AT_T; x += 8)
#pragma unroll
              for (int y = 0; y < 4; ++y)
                m4[y] = fmaxf(fmaxf(m4[y], __uint_as_float(s[x + y])), __uint_as_float(s[x + 4 + y]));
            mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
          }
        }
        const float mn = fmaxf(m, mx * c);
        const bool grow = mn > m + 8.f;
        if (__any_sync(~0u, grow)) {
          const float f = grow ? ex2(m - mn) : 1.f;  // 0 for a row's first visible block
          if (grow) m = mn;
          l *= f;
          if (n > 0) {
            // (16 columns at a time: the scores stay in registers)
#pragma unroll 1
            for (int x = 0; x < DP; x += 16) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(to + x, o);
              tmem_ld_wait();
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
              tmem_st_32x32b_x16(to + x, o);
            }
          }
        }
        const float mm = m == -INFINITY ? 0.f : m;
        float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          uint32_t p[32], lo[EXACT ? 32 : 1];
#pragma unroll
          for (int y = 0; y < 32; ++y) {
            const float p0 = ex2(fmaf(__uint_as_float(s[x * 64 + 2 * y]), c, -mm));
            const float p1 = ex2(fmaf(__uint_as_float(s[x * 64 + 2 * y + 1]), c, -mm));
            l4[2 * (y & 1)] += p0;
            l4[2 * (y & 1) + 1] += p1;
            if constexpr (EXACT)
              parts2<T>(p0, p1, p[y], lo[y]);
            else
              p[y] = pack2<T>(p0, p1);
          }
          tmem_st_32x32b_x32(ts + x * 32, p);
          if constexpr (EXACT) tmem_st_32x32b_x32(ts + 64 + x * 32, lo);
        }
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&p_full[i]);
      }
      if (w.count > 0) {
        ok = ok && at_wait(&o_full[i], no & 1, a.err, abort_flag);
        ++no;
        tc_fence_after();
      }
      if (!(ok = named_all(1 + i, ok))) break;
      const int id = 2 * w.pair + i;
      const int r0 = id / a.G * AT_T, h = w.hk * a.G + id % a.G, row = r0 + rl;
      // which rows see something goes by position (a row sees itself at least),
      // not by their sum, which a NaN or an infinite score makes NaN; a part of a
      // split may have nothing for such a row
      const bool some = row < a.Tq && pr >= 0 && pr < w.len && (!PART || l != 0.f);
      if (a.lse && row < a.Tq)
        a.lse[((int64_t)w.ob * a.Hq + h) * a.Tq + row] = some ? (m + log2f(l)) * AT_LN2 : -INFINITY;
      const float inv = some ? 1.f / l : 0.f;
      if constexpr (PART)
        store_part<DP>(to, so + i * AT_BOX, rl, inv, some, w.count > 0, &tout, a.D, r0, h, w.ob, 1 + i, leader,
                       &o_empty[i]);
      else
        store_tile<T, DP>(to, so + i * AT_BOX, rl, inv, some, w.count > 0, &tout, r0, h, w.ob, 1 + i, leader,
                          &o_empty[i], 0, a.out_lo ? &tlo : nullptr);
    }
    if (leader) bulk_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) tmem_dealloc(tmem, 512);
}

int attn_tmap(CUtensorMap* m, const void* p, int dtype, const Strides3& s, int64_t B, int64_t H, int64_t T, int64_t D,
              int rows) {
  // the stride of a dimension of size 1 is never used, but must be a valid one
  const int size = dtype_size(dtype);
  auto bytes = [&](int64_t st) { return (uint64_t)std::max<int64_t>(st * size, 16); };
  return make_tmap_4d(m, p, dtype, (uint64_t)D, (uint64_t)T, (uint64_t)H, (uint64_t)B, bytes(s.t), bytes(s.h),
                      bytes(s.b), 128u / size, (uint32_t)rows);
}

// The parts of a split joined in their order: 16 lanes a row, as 128-bit pieces.
// Parts are in 32 bits: a part's rounding would come on top of the output's.
// A part whose sum is NaN makes the row NaN (the maximum alone would pass over it).
struct JoinArgs {
  const float* part;  // [splits, B, Hq, Tq, D]
  const float* lse;   // [splits, B, Hq, Tq]
  AttnArgs a;
};
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const JoinArgs j, FastDiv by_t, FastDiv by_h) {
  const AttnArgs& a = j.a;
  const uint32_t r = blockIdx.x * 16u + (threadIdx.x >> 4);
  const uint32_t bh = by_t.div(r), t = r - bh * a.Tq;
  if (bh >= (uint32_t)a.B * a.Hq) return;
  const uint32_t b = by_h.div(bh), h = bh - b * a.Hq;
  const int d = (threadIdx.x & 15) * 8;
  const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
  float m = -INFINITY, sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  bool nan = false;
  for (int s = 0; s < a.splits; ++s) {
    const float e = j.lse[s * rows + r];
    m = fmaxf(m, e);
    nan |= isnan(e);
  }
  const Span sp = attn_span(a.starts, a.ends, (int)b, a.Tk);
  const int p = (int)t + a.Tk - a.Tq;
  const bool real = p >= sp.start && p < sp.end;
  if (real) {
    for (int s = 0; s < a.splits; ++s) {
      const float w = expf(j.lse[s * rows + r] - m);  // (NaN where every score is -inf: 0 / 0)
      sum += w;
      if (d < a.D) {
        float u[8];
        const float4* at = reinterpret_cast<const float4*>(j.part + (s * rows + r) * a.D + d);
        *reinterpret_cast<float4*>(u) = at[0];
        *reinterpret_cast<float4*>(u + 4) = at[1];
#pragma unroll
        for (int y = 0; y < 8; ++y) o[y] = fmaf(w, u[y], o[y]);
      }
    }
    const float inv = 1.f / sum;
#pragma unroll
    for (int y = 0; y < 8; ++y) o[y] *= inv;
  }
  if (d < a.D) {
    const int64_t at = b * a.so.b + h * a.so.h + (int64_t)t * a.so.t + d;
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int y = 0; y < 4; ++y) {
      float f[2];
      hi[y] = pack2<T>(o[2 * y], o[2 * y + 1]);
      unpack2<T>(hi[y], f);
      lo[y] = pack2<T>(o[2 * y] - f[0], o[2 * y + 1] - f[1]);
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    if (a.out_lo) *reinterpret_cast<uint4*>(static_cast<T*>(a.out_lo) + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
  }
  if (a.lse && d == 0) a.lse[r] = !real ? -INFINITY : nan ? NAN : m == -INFINITY ? m : m + logf(sum);
}

bool attn_few_rows(int64_t B, int64_t Hk, int64_t G, int64_t Tq) {
  return Tq * G <= 16 && B <= 65535 && Hk <= 65535;
}

// Where the items are fewer than half the multiprocessors (a chunk of a prompt
// over a long cache), blocks share an item's keys, each with four blocks of
// keys at least, and a second kernel joins them: 501 queries behind 5632 keys,
// 64 items, took 106 us without.
int attn_fwd_splits(int64_t B, int64_t Hk, int64_t G, int64_t Tq, int64_t Tk, int64_t window, int64_t sinks) {
  const int64_t tiles = (Tq + AT_T - 1) / AT_T * G;
  const int64_t items = (tiles + 1) / 2 * B * Hk;
  const int64_t keys = window ? std::min(Tk, std::min(window, Tk) + AT_T + std::min(sinks, Tk)) : Tk;
  return (int)std::max<int64_t>(1, std::min<int64_t>({num_sms() / std::max<int64_t>(items, 1), keys / (4 * AT_T), 16}));
}

// Probabilities and their gradients are rounded to the operands' type for the
// products, u of each value, in effect at random: outputs and gradients are off by
// 1.2 to 1.5 times their own rounding, the most where a row sees few keys, and 1.65
// times where few rows leave the sum to chance as well.  A second product with
// the remainders makes that 1.00, for a third of the time (8192 tokens, forward and
// backward, 1.01 -> 1.32 ms; up to 512 tokens, 55 -> 65 us).  So it is made where few
// keys are seen and at most one tile falls to a multiprocessor, a call bound by
// launches (9 x 128 tokens, 16/8 heads: 37 -> 39 us of kernels, 92 us the call;
// 2 x 24 tokens, 2/1 heads of 32: 26.5 -> 29.8).
bool attn_exact(const AttnArgs& a) {
  const int64_t rows = (int64_t)((a.Tq + AT_T - 1) / AT_T) * a.G;
  const bool few = a.Tk <= AT_T || (a.window && a.window + a.sinks <= 32);
  return few && rows <= 16 && rows * a.B * a.Hk <= num_sms();
}

template <typename T, int DP, FwMode MODE>
static int attn_fwd_go(const AttnArgs& a0, void* workspace, cudaStream_t st) {
  constexpr bool PART = MODE == FW_PART;
  AttnArgs a = a0;
  JoinArgs join{};
  Strides3 so = a.so;
  const int64_t rows = (int64_t)a.B * a.Hq * a.Tq;
  if (PART) {
    // the parts' outputs take the output's place
    join.a = a0;
    a.out = workspace;
    a.out_lo = nullptr;
    join.part = static_cast<const float*>(workspace);
    join.lse = a.lse = static_cast<float*>(workspace) + a.splits * rows * a.D;
    so = Strides3{(int64_t)a.Hq * a.Tq * a.D, (int64_t)a.Tq * a.D, a.D};
  }
  constexpr int dt = DtOf<T>::value;
  // (also makes the device's context current: a tensor map cannot be encoded
  // on a thread that has made no CUDA call yet, such as autograd's)
  if (cudaFuncSetAttribute(attn_fwd_kernel<T, DP, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           FwTile<DP>::SMEM) != cudaSuccess)
    return check_cuda("cudaFuncSetAttribute(attn_fwd)");
  CUtensorMap tq, tk, tv, tout, tlo{};
  int rc;
  if ((rc = attn_tmap(&tq, a.q, dt, a.sq, a.B, a.Hq, a.Tq, a.D)) ||
      (rc = attn_tmap(&tk, a.k, dt, a.sk, a.B, a.Hk, a.Tk, a.D)) ||
      (rc = attn_tmap(&tv, a.v, dt, a.sv, a.B, a.Hk, a.Tk, a.D)) ||
      (rc = attn_tmap(&tout, a.out, PART ? PKM_DT_F32 : dt, so, (int64_t)a.B * a.splits, a.Hq, a.Tq, a.D)) ||
      (a.out_lo && (rc = attn_tmap(&tlo, a.out_lo, dt, so, a.B, a.Hq, a.Tq, a.D))))
    return rc;
  const int64_t tiles = (int64_t)((a.Tq + AT_T - 1) / AT_T) * a.G;
  const int64_t items = (tiles + 1) / 2 * a.B * a.Hk * a.splits;
  if (items > INT32_MAX / 2) return fail(PKM_ERR_UNSUPPORTED, "too many rows");
  const int grid = (int)std::min<int64_t>(items, num_sms());
  attn_fwd_kernel<T, DP, MODE><<<grid, FW_THREADS, FwTile<DP>::SMEM, st>>>(tq, tk, tv, tout, tlo, a);
  if ((rc = check_cuda("attn_fwd")) || !PART) return rc;
  attn_join_kernel<T><<<(unsigned)((rows + 15) / 16), 256, 0, st>>>(join, FastDiv((uint32_t)a.Tq),
                                                                   FastDiv((uint32_t)a.Hq));
  return check_cuda("attn_join");
}

template <typename T, int DP>
static int attn_fwd_parts(const AttnArgs& a, void* workspace, cudaStream_t st) {
  return a.splits > 1    ? attn_fwd_go<T, DP, FW_PART>(a, workspace, st)
         : attn_exact(a) ? attn_fwd_go<T, DP, FW_EXACT>(a, workspace, st)
                         : attn_fwd_go<T, DP, FW_PLAIN>(a, workspace, st);
}

int attn_fwd_launch(const AttnArgs& a, int dtype, void* workspace, cudaStream_t st) {
  if (dtype == PKM_DT_BF16)
    return a.D > 64 ? attn_fwd_parts<__nv_bfloat16, 128>(a, workspace, st)
                    : attn_fwd_parts<__nv_bfloat16, 64>(a, workspace, st);
  return a.D > 64 ? attn_fwd_parts<__half, 128>(a, workspace, st) : attn_fwd_parts<__half, 64>(a, workspace, st);
}

}  // namespace pkm
