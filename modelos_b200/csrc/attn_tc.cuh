// Pieces of the tensor-core attention kernels: tile geometry, descriptors,
// bounded waits, the walk over the blocks that a tile of rows sees.
#pragma once

#include "attn.cuh"
#include "umma.cuh"

namespace pkm {

constexpr int AT_T = 128;                // rows of a query tile, rows of a key block
constexpr int AT_BOX = AT_T * 128;       // bytes of 128 rows x 64 channels
constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr float AT_LN2 = 0.6931471805599453f;

// kind::f16 instruction descriptor, fp32 accumulators, A and B of type `fmt`
// (0 fp16, 1 bf16); b_mn: B is MN-major; a_mn: A is MN-major.
__host__ __device__ constexpr uint32_t at_idesc(int fmt, int M, int N, int a_mn, int b_mn) {
  return (1u << 4) | ((uint32_t)fmt << 7) | ((uint32_t)fmt << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// A tile is 128 rows of up to 128 channels as one or two swizzled boxes of 64
// channels (AT_BOX bytes each).  A shared-memory descriptor is built once per
// tile, as its low and high word; steps add to the low word, the address in
// units of 16 bytes (one thread issues every product, and building whole
// descriptors there took longer than the products: 100 cycles for each of 64).
// Read K-major (channels are the product's K): K step s of 16 channels lies in
// box s / 4.
constexpr uint32_t AT_DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);  // stride, version, 128-byte swizzle
__device__ __forceinline__ uint32_t at_desc_k(uint32_t tile) { return ((tile >> 4) & 0x3fffu) | (1u << 16); }
__device__ __forceinline__ constexpr uint32_t at_step_k(int s) { return ((s >> 2) * AT_BOX + (s & 3) * 32) >> 4; }
// Read MN-major (rows are the product's K): K step s is rows 16 s .. 16 s + 15;
// the channels' blocks of 64 are a box apart.
__device__ __forceinline__ uint32_t at_desc_mn(uint32_t tile) {
  return ((tile >> 4) & 0x3fffu) | ((uint32_t)(AT_BOX >> 4) << 16);
}
__device__ __forceinline__ constexpr uint32_t at_step_mn(int s) { return (s * 2048) >> 4; }

// D (+)= A B^T with both operands in shared memory, or A in TMEM.
template <bool ACC>
__device__ __forceinline__ void at_mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 x, {%1, %3};\n\tmov.b64 y, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(AT_DESC_HI), "r"(idesc), "n"(ACC ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void at_mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\t"
      "setp.ne.b32 p, %5, 0;\n\tmov.b64 y, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %4, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(AT_DESC_HI), "r"(idesc), "r"(acc)
      : "memory");
}
// The products of a whole tile: S = A B^T over DP channels; D += P B over the
// 128 rows of B, P in TMEM, its second 64 columns GAP columns behind the
// first 32 (two values a column).
template <int DP>
__device__ __forceinline__ void at_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  at_mma_ss<false>(d, a, b, idesc);
#pragma unroll
  for (int s = 1; s < DP / 16; ++s) at_mma_ss<true>(d, a + at_step_k(s), b + at_step_k(s), idesc);
}
template <int GAP>
__device__ __forceinline__ void at_accum(uint32_t d, uint32_t p, uint32_t b, uint32_t idesc, bool first) {
  at_mma_ts(d, p, b, idesc, first ? 0u : 1u);
#pragma unroll
  for (int s = 1; s < AT_T / 16; ++s)
    at_mma_ts(d, p + (s >> 2) * GAP + (s & 3) * 8, b + at_step_mn(s), idesc, 1u);
}

// Bounded wait on an mbarrier; the first role that gives up sets the abort
// flag and the others leave.
__device__ __forceinline__ bool at_wait(uint64_t* bar, uint32_t parity, uint32_t* err, volatile int* abort_flag) {
  for (uint32_t i = 0; i < kWaitLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 1023) == 1023 && *abort_flag) return false;
  }
  raise_err(err, PKM_DEVERR_TIMEOUT);
  *abort_flag = 1;
  return false;
}

// A block whose last rows lie behind the sequence (they may hold anything, NaN
// included) arrives on a barrier of its own, `landed`; one warp zeroes rows
// [rem, 128) for the products that read the tile through the async proxy, and
// then arrives on the barrier `full` that the products wait for.
template <int DP>
__device__ __forceinline__ bool zero_tail(unsigned char* tile, int rem, int lane, uint64_t* landed, uint32_t parity,
                                          uint64_t* full, uint32_t* err, volatile int* abort_flag) {
  const bool got = at_wait(landed, parity, err, abort_flag);
  if (!__all_sync(~0u, got)) return false;
  for (int r = rem * 8 + lane; r < AT_T * 8; r += 32)
    for (int x = 0; x < DP / 64; ++x) *reinterpret_cast<uint4*>(tile + x * AT_BOX + r * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) mbar_arrive(full);
  return true;
}

// Every warp of a warpgroup executes one of these.
template <int N>
__device__ __forceinline__ void reg_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void reg_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float (&f)[2]);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float (&f)[2]) {
  f[0] = __uint_as_float(w << 16);
  f[1] = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float (&f)[2]) {
  const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w));
  f[0] = t.x;
  f[1] = t.y;
}

// What packing (x, y) to w left, packed.
template <typename T>
__device__ __forceinline__ uint32_t remainder2(float x, float y, uint32_t w) {
  float f[2];
  unpack2<T>(w, f);
  return pack2<T>(x - f[0], y - f[1]);
}

// Probabilities (not negative) as two packed parts for two products.  The first is
// rounded towards 0, so that the second is not negative, and where the first is
// not 0 the second is at least the type's smallest number: times an infinite value
// both parts are that infinity, and their sum is not NaN.
template <typename T>
__device__ __forceinline__ uint32_t pack2_down(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2_down<__nv_bfloat16>(float x, float y) {
  uint32_t w;
  asm("cvt.rz.bf16x2.f32 %0, %2, %1;" : "=r"(w) : "f"(x), "f"(y));
  return w;
}
template <>
__device__ __forceinline__ uint32_t pack2_down<__half>(float x, float y) {
  uint32_t w;
  asm("cvt.rz.f16x2.f32 %0, %2, %1;" : "=r"(w) : "f"(x), "f"(y));
  return w;
}
template <typename T>
__device__ __forceinline__ void parts2(float x, float y, uint32_t& first, uint32_t& second) {
  first = pack2_down<T>(x, y);
  second = __vmaxu2(remainder2<T>(x, y, first), __vsetne2(first, 0u));
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Tensor map over [B, H, T, D] with boxes of 128 bytes of channels x `rows` tokens.
int attn_tmap(CUtensorMap* m, const void* p, int dtype, const Strides3& s, int64_t B, int64_t H, int64_t T, int64_t D,
              int rows = AT_T);

// Bits of the columns x0 .. x0 + 31 with x <= top and (x >= low or x < sink).
__device__ __forceinline__ uint32_t upto(int n) { return n < 0 ? 0u : 0xffffffffu >> (31 - min(n, 31)); }
__device__ __forceinline__ uint32_t seen_bits(int x0, int top, int low, int sink) {
  return upto(top - x0) & (~upto(low - 1 - x0) | upto(sink - 1 - x0));
}

// Blocks of a walk: `head` blocks from 0, then up to `last` from `from` on.
// Blocks are counted from the sequence's first row, so that its front edge
// never lies inside a block.
struct Walk {
  int head, from, count;
  __device__ __forceinline__ int block(int n) const { return n < head ? n : from + (n - head); }
};

// Key blocks that the query rows [p0, p1] (relative to the sequence's start,
// length `len`) see.
__device__ __forceinline__ void at_key_range(int p0, int p1, int len, int window, int& lo, int& hi) {
  p0 = max(p0, 0);
  p1 = min(p1, len - 1);
  if (p0 > p1) {
    lo = INT32_MAX;
    hi = 0;
    return;
  }
  hi = p1 / AT_T + 1;
  lo = window ? max(0, p0 - window + 1) / AT_T : 0;
}
__device__ __forceinline__ Walk at_key_walk(int lo, int hi, int sinks) {
  Walk w;
  if (hi == 0) {
    w.head = w.from = w.count = 0;
    return w;
  }
  const int ns = min((sinks + AT_T - 1) / AT_T, hi);
  w.head = lo <= ns ? 0 : ns;
  w.from = lo <= ns ? (ns > 0 ? 0 : lo) : lo;
  w.count = w.head + hi - w.from;
  return w;
}

// The work items of one block of a persistent grid: items are in order of
// falling work, and blocks take them forwards and backwards in turn, so that
// each gets about the same sum.
struct Items {
  int count, k;
  __device__ __forceinline__ explicit Items(int n) : count(n), k(0) {}
  __device__ __forceinline__ bool next(int& item) {
    const int g = (int)gridDim.x;
    item = k * g + ((k & 1) ? g - 1 - (int)blockIdx.x : (int)blockIdx.x);
    ++k;
    return item < count;
  }
};

// 128 threads (named barrier `id`) store a tile of accumulator rows times `f`
// (zeros where !some) as 128 x DP of T: 64 channels at a time through a
// swizzled box in shared memory and a TMA store.  (Stores of a row a thread
// took 5700 cycles for a tile, one row's sector at a time.)  With `lo`, what
// the rounding left is stored too.  The thread with `leader` set keeps the
// stores' group; `have`: there are accumulators.  `drained` is arrived on once
// the accumulators are read.
__device__ __forceinline__ void named_sync(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// Whether `ok` holds for all 128 threads of a group: a group leaves together,
// or some of it would wait for the rest at a named barrier.
__device__ __forceinline__ bool named_all(int id, bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
      "bar.red.and.pred p, %1, 128, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "r"(id), "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <typename T, int DP>
__device__ __forceinline__ void store_tile(uint32_t taddr, unsigned char* box, int row, float f, bool some, bool have,
                                           const CUtensorMap* map, int y, int z, int w, int id, bool leader,
                                           uint64_t* drained, int x0 = 0, const CUtensorMap* lo = nullptr) {
  const uint32_t sb = smem_u32(box) + row * 128;
  const int parts = lo ? 2 : 1;
  // (loops that stay loops: with them unrolled, the compiler spills the
  // registers of the code before, which took twice its time)
#pragma unroll 1
  for (int x = 0; x < DP; x += 64) {
#pragma unroll 1
    for (int part = 0; part < parts; ++part) {
      if (leader) bulk_wait_read_all();  // the box's last contents have left
      named_sync(id, AT_T);
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        uint32_t o[32];
        if (have) {
          tmem_ld_32x32b_x32(taddr + x + half * 32, o);
          tmem_ld_wait();
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[4] = {0, 0, 0, 0};
          if (have && some) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float u = __uint_as_float(o[c * 8 + 2 * e]) * f, t = __uint_as_float(o[c * 8 + 2 * e + 1]) * f;
              v[e] = pack2<T>(u, t);
              if (part) {
                float r[2];
                unpack2<T>(v[e], r);
                v[e] = pack2<T>(u - r[0], t - r[1]);
              }
            }
          }
          sts128(sb + (((half * 4 + c) ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
        }
      }
      if (have && x + 64 == DP && part + 1 == parts) {
        tc_fence_before();
        mbar_arrive(drained);
      }
      fence_proxy_async_smem();
      named_sync(id, AT_T);
      if (leader) {
        tma_store_4d(part ? lo : map, box, x0 + x, y, z, w);
        bulk_commit_group();
      }
    }
  }
}

// The same for a partial result, in 32 bits: 32 channels at a time, up to the
// last of the tensor's D (a box starts inside the tensor).
template <int DP>
__device__ __forceinline__ void store_part(uint32_t taddr, unsigned char* box, int row, float f, bool some, bool have,
                                           const CUtensorMap* map, int D, int y, int z, int w, int id, bool leader,
                                           uint64_t* drained) {
  const uint32_t sb = smem_u32(box) + row * 128;
  const int channels = min(D, DP);
#pragma unroll 1
  for (int x = 0; x < channels; x += 32) {
    if (leader) bulk_wait_read_all();
    named_sync(id, AT_T);
    uint32_t o[32];
    if (have) {
      tmem_ld_32x32b_x32(taddr + x, o);
      tmem_ld_wait();
      if (x + 32 >= channels) {
        tc_fence_before();
        mbar_arrive(drained);
      }
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t v[4] = {0, 0, 0, 0};
      if (have && some) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __float_as_uint(__uint_as_float(o[c * 4 + e]) * f);
      }
      sts128(sb + ((c ^ (row & 7)) << 4), v[0], v[1], v[2], v[3]);
    }
    fence_proxy_async_smem();
    named_sync(id, AT_T);
    if (leader) {
      tma_store_4d(map, box, x, y, z, w);
      bulk_commit_group();
    }
  }
}

}  // namespace pkm
