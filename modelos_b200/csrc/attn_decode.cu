// Attention of few query rows over many keys (single tokens of a cached
// decode, a few tokens at once), keys and values in 16 bits or in the 4-bit
// cache.  Bound by the bytes of the visible keys and values.
//
// A block serves one sequence's key/value head and 8 * NT of its query rows
// (tokens x grouped heads), and a part of the visible keys: a cluster of
// `splits` blocks shares them and joins its partial results through
// distributed shared memory, so that there is one launch and no workspace.
//   producer warp  TMA (16 bits) or bulk copies (4-bit codes, plus
//                  cp.async for their steps and offsets) into a ring;
//   other warps    16 keys of each stage per warp, mma.sync m16n8k16 with
//                  the keys (channels) as the 16 rows and the query rows as
//                  the 8 columns:  S^T = K Q^T,  O^T += V^T P^T.
// The tensor instructions here are the small ones on purpose: 8 query rows
// fill them, the tcgen05 tiles of 128 rows would be 6 % full, and the time
// goes to the copies.  The running maximum of a row is raised only when a
// score exceeds it by more than 2^8 (which a vote finds without reducing).
//
// Measured (16/8 heads of 128, bf16): 32 sequences with 8196 visible keys, 157 us
// (6.8 TB/s, at the memory's rate); 8 with 2305, 12.8 us (5.9 TB/s).  4 bits, 32
// sequences of 14100 to 16000 keys: 169 us (3.6 TB/s), bound by instructions: 428
// for 16 keys, 240 of them make codes into values.
//
// 4 bits: two keys' codes are interleaved before they become values, so that
// a register holds the pair of keys that an operand of O^T += V^T P^T needs.
#include <algorithm>
#include <atomic>

#include "attn_tc.cuh"
#include "kv4.cuh"

namespace pkm {

constexpr int DC_ROWS = 8;  // query rows of an n tile

struct DecodeArgs {
  const void* q;
  Strides3 sq;
  void* out;
  void* out_lo;
  Strides3 so;
  float* lse;
  const uint8_t* codes[2];
  const void* params[2];
  int B, Hq, Hk, G, Tq, rows, D, splits;  // rows: of keys (Tk or the cache's capacity)
  int own_end;                            // queries are a sequence's last rows (else the tensor's)
  float scale;
  int window, sinks;
  const int32_t* starts;
  const int32_t* ends;
  uint32_t* err;
};

template <int DP, int NT, bool Q4>
struct DecodeTile {
  static constexpr int WARPS = 4;
  static constexpr int SUB = Q4 ? 2 : 1;  // 16-key parts a warp takes of a stage
  static constexpr int KEYS = 16 * SUB * WARPS;
  static constexpr int THREADS = 32 * (WARPS + 1);
  static constexpr int SIDE = Q4 ? KEYS * DP / 2 : KEYS * DP * 2;  // codes or values of a stage
  static constexpr int PAR = Q4 ? KEYS * (DP / 32) * 4 : 0;
  static constexpr int STAGE = 2 * (SIDE + PAR);
  static constexpr int STAGES = Q4 ? (DP == 128 ? 2 : 4) : (DP == 128 ? 3 : 5);
  static constexpr int BLOCKS = Q4 ? (NT == 1 ? 4 : 3) : 2;  // to a multiprocessor
  static constexpr int ROWS = DC_ROWS * NT;
  static constexpr int SLAB = ROWS * DP * 4;  // a warp's partial result
  static constexpr int RING = STAGES * STAGE > WARPS * SLAB ? STAGES * STAGE : WARPS * SLAB;
  static constexpr int SMEM = RING + SLAB + (2 * WARPS + 2) * ROWS * 4 + 2 * STAGES * 8 + 16 + 1024;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// The keys that some of the rows sees, as stages: sink tokens that lie before
// the window, then the window.
struct DecodeKeys {
  int start, end, head, from, head_stages, stages;
  __device__ __forceinline__ void stage(int u, int keys, int& row, int& count) const {
    if (u < head_stages) {
      row = start + u * keys;
      count = min(keys, head - u * keys);
    } else {
      row = from + (u - head_stages) * keys;
      count = min(keys, end - row);
    }
  }
};

template <typename T, int DP, int NT, bool Q4>
__global__ void __launch_bounds__(DecodeTile<DP, NT, Q4>::THREADS, DecodeTile<DP, NT, Q4>::BLOCKS)
    attn_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const DecodeArgs a) {
  using F = DecodeTile<DP, NT, Q4>;
  constexpr int KS = DP / 16;     // K steps of S^T, and d tiles of O^T
  constexpr int PB = DP / 32 * 4;  // bytes of a token's steps and offsets
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                                         ~static_cast<uintptr_t>(1023));
  float* block_o = reinterpret_cast<float*>(smem + F::RING);  // [ROWS][DP]
  float* block_m = block_o + F::ROWS * DP;                    // [ROWS]
  float* block_l = block_m + F::ROWS;
  float* warp_m = block_l + F::ROWS;  // [WARPS][ROWS]
  float* warp_l = warp_m + F::WARPS * F::ROWS;
  uint64_t* full = reinterpret_cast<uint64_t*>(warp_l + F::WARPS * F::ROWS);
  uint64_t* empty = full + F::STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(empty + F::STAGES);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, hk = blockIdx.y % a.Hk, group = blockIdx.y / a.Hk, b = blockIdx.z;
  const Span sp = attn_span(a.starts, a.ends, b, a.rows);
  const int R = a.Tq * a.G;                       // query rows of this head, G to a token
  const int base = (a.own_end ? sp.end : a.rows) - a.Tq;  // row of the first query token
  const int row0 = group * F::ROWS;
  const int rows = min(F::ROWS, R - row0);
  const int p_first = base + row0 / a.G, p_last = base + (row0 + rows - 1) / a.G;

  DecodeKeys keys;
  {
    // queries outside the sequence see nothing
    const int p0 = max(p_first, sp.start), p1 = min(p_last, sp.end - 1);
    keys.start = sp.start;
    keys.end = p0 <= p1 ? p1 + 1 : sp.start;
    keys.from = a.window ? max(sp.start, p0 - a.window + 1) : sp.start;
    const int sink_end = a.window ? min(sp.start + a.sinks, keys.end) : sp.start;
    if (p0 > p1) keys.from = sp.start;
    keys.head = keys.from > sink_end ? sink_end - sp.start : 0;
    if (keys.from <= sink_end) keys.from = sp.start;
    keys.head_stages = (keys.head + F::KEYS - 1) / F::KEYS;
    keys.stages = keys.head_stages + (max(keys.end - keys.from, 0) + F::KEYS - 1) / F::KEYS;
  }
  const int u0 = (int)((int64_t)keys.stages * split / a.splits);
  const int u1 = (int)((int64_t)keys.stages * (split + 1) / a.splits);

  if (threadIdx.x == 0) {
    for (int i = 0; i < F::STAGES; ++i) {
      mbar_init(&full[i], Q4 ? 33 : 1);
      mbar_init(&empty[i], F::WARPS);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  __syncthreads();

  if (warp == F::WARPS) {
    int u = u0;
    for (; u < u1; ++u) {
      const int n = u - u0, st = n % F::STAGES;
      const bool got = at_wait(&empty[st], ((n / F::STAGES) & 1) ^ 1, a.err, abort_flag);
      if (!__all_sync(~0u, got)) break;
      int row, count;
      keys.stage(u, F::KEYS, row, count);
      unsigned char* buf = smem + st * F::STAGE;
      if constexpr (Q4) {
        const int64_t slot = (int64_t)(b * a.Hk + hk) * a.rows + row;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[st], 2 * count * (DP / 2));
          bulk_g2s(buf, a.codes[0] + slot * (DP / 2), count * (DP / 2), &full[st]);
          bulk_g2s(buf + F::SIDE, a.codes[1] + slot * (DP / 2), count * (DP / 2), &full[st]);
        }
#pragma unroll
        for (int side = 0; side < 2; ++side) {
          const unsigned char* src = static_cast<const unsigned char*>(a.params[side]) + slot * PB;
          const uint32_t dst = smem_u32(buf + 2 * F::SIDE + side * F::PAR);
          for (int r = lane; r < count; r += 32)
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst + r * PB), "l"(src + r * PB), "n"(PB)
                         : "memory");
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
      } else if (lane == 0) {
        mbar_arrive_expect_tx(&full[st], 2 * F::SIDE);
        for (int x = 0; x < DP / 64; ++x) {
          tma_load_4d(buf + x * (F::KEYS * 128), &tk, x * 64, row, hk, b, &full[st]);
          tma_load_4d(buf + F::SIDE + x * (F::KEYS * 128), &tv, x * 64, row, hk, b, &full[st]);
        }
      }
    }
    // copies in flight land before the ring is used for something else
    for (int n = max(0, u - u0 - F::STAGES); n < u - u0; ++n)
      mbar_wait(&full[n % F::STAGES], (n / F::STAGES) & 1, nullptr);
  } else {
    const int g = lane >> 2, t = lane & 3;
    const float c = a.scale * AT_LOG2E;
    // Q^T as B operands: query row g of each n tile, this lane's channels
    uint32_t qb[NT][KS][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * DC_ROWS + g;
      const T* qp = static_cast<const T*>(a.q) + b * a.sq.b + (int64_t)(hk * a.G + r % a.G) * a.sq.h +
                    (int64_t)(r / a.G) * a.sq.t;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (Q4) {
          // word s / 2 of this lane's codes: pairs of channels (j, j + 4), j = 2 (s & 1) and the next
          const int d = t * (DP / 4) + (s >> 1) * 8 + (s & 1) * 2;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            uint32_t w = 0;
            if (r < R) {
              const uint16_t x0 = reinterpret_cast<const uint16_t*>(qp)[d + y];
              const uint16_t x1 = reinterpret_cast<const uint16_t*>(qp)[d + y + 4];
              w = (uint32_t)x0 | ((uint32_t)x1 << 16);
            }
            qb[nt][s][y] = w;
          }
        } else {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int d = s * 16 + y * 8 + 2 * t;
            qb[nt][s][y] = r < R && d < a.D ? *reinterpret_cast<const uint32_t*>(qp + d) : 0u;
          }
        }
      }
    }
    float o[NT][KS][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) o[nt][s][0] = o[nt][s][1] = o[nt][s][2] = o[nt][s][3] = 0.f;
    }
    // key of 16 that row g of the instruction stands for (4 bits: so that a
    // lane's four keys of V lie 4 tokens apart)
    const int kg = Q4 ? (g >> 1) + (g & 1) * 4 : g;
    int pos[NT][2];  // positions of this lane's query rows
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const int p = base + (row0 + nt * DC_ROWS + 2 * t + y) / a.G;
        pos[nt][y] = p < sp.end ? p : -1;
      }
    const uint32_t ring = smem_u32(smem);
    constexpr int W = DP / 32;  // words of codes a lane takes from a key of K, twice those of V

    int st = 0;
    uint32_t ph = 0;
    for (int u = u0; u < u1; ++u) {
      const bool got = at_wait(&full[st], ph, a.err, abort_flag);
      if (!__all_sync(~0u, got)) break;
      int row, count;
      keys.stage(u, F::KEYS, row, count);
      const int k0 = warp * (16 * F::SUB);
      const int left = count - k0;  // this warp's keys
      if (left > 0) {
        const uint32_t buf = ring + st * F::STAGE;
        float x[F::SUB][NT][4];
#pragma unroll
        for (int sub = 0; sub < F::SUB; ++sub) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) x[sub][nt][0] = x[sub][nt][1] = x[sub][nt][2] = x[sub][nt][3] = 0.f;
          // ---- S^T = K Q^T
          if constexpr (Q4) {
            uint32_t w0[W], w1[W];
            const int key = k0 + sub * 16 + kg;
            const uint32_t c0 = buf + key * (DP / 2) + t * (DP / 8);
            if constexpr (W == 4) {
              const uint4 v0 = lds128(c0), v1 = lds128(c0 + 8 * (DP / 2));
              w0[0] = v0.x, w0[1] = v0.y, w0[2] = v0.z, w0[3] = v0.w;
              w1[0] = v1.x, w1[1] = v1.y, w1[2] = v1.z, w1[3] = v1.w;
            } else {
              const uint2 v0 = lds64(c0), v1 = lds64(c0 + 8 * (DP / 2));
              w0[0] = v0.x, w0[1] = v0.y, w1[0] = v1.x, w1[1] = v1.y;
            }
            const uint32_t pp = buf + 2 * F::SIDE + key * PB + (DP == 128 ? t : t >> 1) * 4;
            const uint32_t e0 = lds32(pp), e1 = lds32(pp + 8 * PB);
            const uint32_t s0 = __byte_perm(e0, e0, 0x1010), f0 = __byte_perm(e0, e0, 0x3232);
            const uint32_t s1 = __byte_perm(e1, e1, 0x1010), f1 = __byte_perm(e1, e1, 0x3232);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              const int sh = (s & 1) * 8;
              const uint32_t r[4] = {
                  dequant2<T>(w0[s >> 1] >> sh, s0, f0), dequant2<T>(w1[s >> 1] >> sh, s1, f1),
                  dequant2<T>(w0[s >> 1] >> (sh + 4), s0, f0), dequant2<T>(w1[s >> 1] >> (sh + 4), s1, f1)};
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<T>(x[sub][nt], r, qb[nt][s][0], qb[nt][s][1]);
            }
          } else {
            const int kr = k0 + sub * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
            const uint32_t kb = buf + kr * 128;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              uint32_t r[4];
              const int ch = (s & 3) * 2 + (lane >> 4);
              ldsm4(r, kb + (s >> 2) * (F::KEYS * 128) + ((ch ^ (lane & 7)) << 4));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816<T>(x[sub][nt], r, qb[nt][s][0], qb[nt][s][1]);
            }
          }
        }
        // ---- softmax: this lane has keys kg, kg + 8 of query rows 2t, 2t + 1
        const int j = row + k0;
        constexpr int MINE = 16 * F::SUB;
        const bool whole = left >= MINE && j + MINE - 1 <= p_first && p_last < sp.end &&
                           (a.window == 0 || j > p_last - a.window || j + MINE <= sp.start + a.sinks);
        bool raise = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int sub = 0; sub < F::SUB; ++sub)
#pragma unroll
            for (int y = 0; y < 4; ++y) x[sub][nt][y] *= c;
          if (!whole) {
#pragma unroll
            for (int sub = 0; sub < F::SUB; ++sub)
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                const int p = pos[nt][y & 1], k = sub * 16 + kg + (y >> 1) * 8, kj = j + k;
                const bool see =
                    k < left && kj <= p && (a.window == 0 || kj > p - a.window || kj < sp.start + a.sinks);
                if (!see) x[sub][nt][y] = -INFINITY;
              }
          }
          float mx[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            mx[y] = fmaxf(x[0][nt][y], x[0][nt][y + 2]);
            if constexpr (F::SUB == 2) mx[y] = fmaxf(mx[y], fmaxf(x[1][nt][y], x[1][nt][y + 2]));
          }
          raise |= mx[0] > m[nt][0] + 8.f || mx[1] > m[nt][1] + 8.f;
        }
        if (__any_sync(~0u, raise)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              float mx = fmaxf(x[0][nt][y], x[0][nt][y + 2]);
              if constexpr (F::SUB == 2) mx = fmaxf(mx, fmaxf(x[1][nt][y], x[1][nt][y + 2]));
#pragma unroll
              for (int d = 4; d < 32; d <<= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, d));
              const float mn = fmaxf(m[nt][y], mx);
              const float f = mn == -INFINITY ? 1.f : ex2(m[nt][y] - mn);
              m[nt][y] = mn;
              l[nt][y] *= f;
#pragma unroll
              for (int s = 0; s < KS; ++s) {
                o[nt][s][y] *= f;
                o[nt][s][y + 2] *= f;
              }
            }
          }
        }
        // Probabilities in the keys' type for the product.  16 bits: with what
        // their rounding left as a second product, without which the output's error
        // was 1.3 times that of its own rounding; the copies are what bounds the
        // kernel (8196 keys, 32 sequences: 156 -> 157 us; 2305 keys, 8: 12.2 -> 12.8).
        // 4 bits: bound by instructions, and the codes' error is many times larger.
        uint32_t pb[F::SUB][NT][2], pl[F::SUB][NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float ma = m[nt][0] == -INFINITY ? 0.f : m[nt][0], mb = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
          for (int sub = 0; sub < F::SUB; ++sub) {
            const float p0 = ex2(x[sub][nt][0] - ma), p1 = ex2(x[sub][nt][1] - mb);
            const float p2 = ex2(x[sub][nt][2] - ma), p3 = ex2(x[sub][nt][3] - mb);
            l[nt][0] += p0 + p2;
            l[nt][1] += p1 + p3;
            uint32_t h[2], r[2];
            if constexpr (Q4) {
              h[0] = pack2<T>(p0, p1);
              h[1] = pack2<T>(p2, p3);
            } else {
              parts2<T>(p0, p1, h[0], r[0]);
              parts2<T>(p2, p3, h[1], r[1]);
              pl[sub][nt][0] = transpose8x8(r[0]);
              pl[sub][nt][1] = transpose8x8(r[1]);
            }
            pb[sub][nt][0] = transpose8x8(h[0]);
            pb[sub][nt][1] = transpose8x8(h[1]);
          }
        }
        // ---- O^T += V^T P^T; keys behind the stage's count may hold anything
        // and become zeros (4 bits: by a step and an offset of 0)
#pragma unroll
        for (int sub = 0; sub < F::SUB; ++sub) {
          if constexpr (Q4) {
            uint32_t w[4][W / 2], e[4], step[2], off[2];
            const int key = k0 + sub * 16 + t;
            const uint32_t vc = buf + F::SIDE + key * (DP / 2) + g * (DP / 16);
            const uint32_t vp = buf + 2 * F::SIDE + F::PAR + key * PB + (DP == 128 ? g >> 1 : g >> 2) * 4;
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              if constexpr (W == 4) {
                const uint2 v = lds64(vc + y * 4 * (DP / 2));
                w[y][0] = v.x, w[y][1] = v.y;
              } else {
                w[y][0] = lds32(vc + y * 4 * (DP / 2));
              }
              e[y] = lds32(vp + y * 4 * PB);
              if (sub * 16 + t + y * 4 >= left) e[y] = 0;
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              step[y] = __byte_perm(e[2 * y], e[2 * y + 1], 0x5410);
              off[y] = __byte_perm(e[2 * y], e[2 * y + 1], 0x7632);
            }
#pragma unroll
            for (int i = 0; i < W / 2; ++i) {
              uint32_t lo[2], hi[2];
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                lo[y] = __byte_perm(w[2 * y][i], w[2 * y + 1][i], 0x5410);
                hi[y] = __byte_perm(w[2 * y][i], w[2 * y + 1][i], 0x7632);
              }
#pragma unroll
              for (int z = 0; z < 4; ++z) {
                const uint32_t r[4] = {dequant2<T>(lo[0] >> (4 * z), step[0], off[0]),
                                       dequant2<T>(hi[0] >> (4 * z), step[0], off[0]),
                                       dequant2<T>(lo[1] >> (4 * z), step[1], off[1]),
                                       dequant2<T>(hi[1] >> (4 * z), step[1], off[1])};
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][i * 4 + z], r, pb[sub][nt][0], pb[sub][nt][1]);
              }
            }
          } else {
            const int kr = k0 + sub * 16 + (lane >> 4) * 8 + (lane & 7), rest = left - sub * 16;
            const uint32_t vb = buf + F::SIDE + kr * 128;
            const uint32_t keep0 = (2 * t < rest ? 0xffffu : 0u) | (2 * t + 1 < rest ? 0xffff0000u : 0u);
            const uint32_t keep1 = (2 * t + 8 < rest ? 0xffffu : 0u) | (2 * t + 9 < rest ? 0xffff0000u : 0u);
            // (a tile's second product a step later, so as not to wait for its first)
            uint32_t r[2][4];
#pragma unroll
            for (int s = 0; s <= KS; ++s) {
              if (s < KS) {
                uint32_t(&v)[4] = r[s & 1];
                const int ch = (s & 3) * 2 + ((lane >> 3) & 1);
                ldsm4t(v, vb + (s >> 2) * (F::KEYS * 128) + ((ch ^ (lane & 7)) << 4));
                if (rest < 16) {
                  v[0] &= keep0;
                  v[1] &= keep0;
                  v[2] &= keep1;
                  v[3] &= keep1;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][s], v, pb[sub][nt][0], pb[sub][nt][1]);
              }
              if (s > 0)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
                  mma16816<T>(o[nt][s - 1], r[(s - 1) & 1], pl[sub][nt][0], pl[sub][nt][1]);
            }
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
      if (++st == F::STAGES) {
        st = 0;
        ph ^= 1u;
      }
    }
    // the row's sum over the lanes that share it
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][y] += __shfl_xor_sync(~0u, l[nt][y], d);
        if (g == 0) {
          warp_m[warp * F::ROWS + nt * DC_ROWS + 2 * t + y] = m[nt][y];
          warp_l[warp * F::ROWS + nt * DC_ROWS + 2 * t + y] = l[nt][y];
        }
      }
    // the ring is free once every warp and every copy is done with it
    __syncthreads();
    float* slab = reinterpret_cast<float*>(smem) + warp * (F::ROWS * DP);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int d = Q4 ? g * (DP / 8) + (s >> 2) * 8 + (y >> 1) * 4 + (s & 3) : s * 16 + (y >> 1) * 8 + g;
          slab[(nt * DC_ROWS + 2 * t + (y & 1)) * DP + d] = o[nt][s][y];
        }
  }
  if (warp == F::WARPS) __syncthreads();
  __syncthreads();
  // join the warps, in their order
  for (int e = threadIdx.x; e < F::ROWS * DP; e += F::THREADS) {
    const int r = e / DP;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < F::WARPS; ++w) mx = fmaxf(mx, warp_m[w * F::ROWS + r]);
    float sum = 0.f, ls = 0.f;
    // (a warp without anything for the row has a sum of 0; one with a NaN score
    // has a NaN, which the maximum does not show)
#pragma unroll
    for (int w = 0; w < F::WARPS; ++w) {
      const float lw = warp_l[w * F::ROWS + r];
      if (lw != 0.f) {
        const float f = ex2(warp_m[w * F::ROWS + r] - mx);
        sum = fmaf(f, reinterpret_cast<const float*>(smem)[w * F::ROWS * DP + e], sum);
        ls = fmaf(f, lw, ls);
      }
    }
    block_o[e] = sum;
    if (e % DP == 0) {
      block_m[r] = mx;
      block_l[r] = ls;
    }
  }
  // join the splits, each block of the cluster a part of the rows and channels
  __syncwarp();
  if (a.splits > 1)
    cluster_sync_all();
  else
    __syncthreads();
  const int S = a.splits;
  const uint32_t om = smem_u32(block_o), mm = smem_u32(block_m), lm = smem_u32(block_l);
  for (int e = split * F::THREADS + threadIdx.x; e < rows * (DP / 2); e += S * F::THREADS) {
    const int r = e / (DP / 2), d = e % (DP / 2) * 2;
    float mx = -INFINITY, sum = 0.f, x0 = 0.f, x1 = 0.f;
    if (S == 1) {
      mx = block_m[r];
      sum = block_l[r];
      x0 = block_o[r * DP + d];
      x1 = block_o[r * DP + d + 1];
    } else {
      for (int s = 0; s < S; ++s) mx = fmaxf(mx, ld_cluster(mapa_shared(mm + r * 4, s)));
      for (int s = 0; s < S; ++s) {
        const float ls = ld_cluster(mapa_shared(lm + r * 4, s));
        if (ls == 0.f) continue;
        const float f = ex2(ld_cluster(mapa_shared(mm + r * 4, s)) - mx);
        const uint32_t p = mapa_shared(om + (r * DP + d) * 4, s);
        sum = fmaf(f, ls, sum);
        x0 = fmaf(f, ld_cluster(p), x0);
        x1 = fmaf(f, ld_cluster(p + 4), x1);
      }
    }
    const int qr = row0 + r, i = qr / a.G, h = hk * a.G + qr % a.G;
    // a row of the sequence sees itself at least; its sum is 0 or NaN only if its scores are -inf or NaN
    const bool real = base + i >= sp.start && base + i < sp.end;
    const float inv = 1.f / sum;
    if (d < a.D) {
      const int64_t at = b * a.so.b + h * a.so.h + (int64_t)i * a.so.t + d;
      const uint32_t hi = real ? pack2<T>(x0 * inv, x1 * inv) : 0u;
      *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + at) = hi;
      if (a.out_lo) {
        float f[2];
        unpack2<T>(hi, f);
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out_lo) + at) =
            real ? pack2<T>(x0 * inv - f[0], x1 * inv - f[1]) : 0u;
      }
    }
    if (a.lse && d == 0)
      a.lse[((int64_t)b * a.Hq + h) * a.Tq + i] = real ? (mx + log2f(sum)) * AT_LN2 : -INFINITY;
  }
  __syncwarp();
  if (a.splits > 1) cluster_sync_all();  // the others read this block's shared memory until here
}

// Blocks a cluster shares a head's keys over: the number whose waves over the
// GPU's slots, each a block's stages plus what starting and joining it cost
// (about three stages), are the shortest; clusters of 16 (not portable) only
// where 8 leave multiprocessors without a block.
static int decode_splits(int64_t heads, int64_t stages, int64_t slots, int64_t sms) {
  int best = 1;
  int64_t least = INT64_MAX;
  for (int s = 1; s <= 16 && s <= std::max<int64_t>(stages, 1); s *= 2) {
    if (s == 16 && heads * 8 >= sms) break;
    const int64_t waves = (heads * s + slots - 1) / slots;
    const int64_t t = waves * ((stages + s - 1) / s + 3);
    if (t < least) {
      least = t;
      best = s;
    }
  }
  return best;
}

template <typename T, int DP, int NT, bool Q4>
static int decode_go(DecodeArgs a, const AttnArgs* dense, int64_t visible, cudaStream_t st) {
  using F = DecodeTile<DP, NT, Q4>;
  auto kern = attn_decode_kernel<T, DP, NT, Q4>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM) != cudaSuccess)
    return check_cuda("cudaFuncSetAttribute(attn_decode)");
  CUtensorMap tk{}, tv{};
  if (!Q4) {
    constexpr int dt = DtOf<T>::value;
    int rc;
    if ((rc = attn_tmap(&tk, dense->k, dt, dense->sk, a.B, a.Hk, a.rows, a.D, F::KEYS)) ||
        (rc = attn_tmap(&tv, dense->v, dt, dense->sv, a.B, a.Hk, a.rows, a.D, F::KEYS)))
      return rc;
  }
  const int groups = (a.Tq * a.G + F::ROWS - 1) / F::ROWS;
  const int64_t heads = (int64_t)a.B * a.Hk * groups;
  if (a.B > 65535 || (int64_t)a.Hk * groups > 65535) return fail(PKM_ERR_UNSUPPORTED, "more than 65535 sequences");
  a.splits = decode_splits(heads, (visible + F::KEYS - 1) / F::KEYS, (int64_t)num_sms() * F::BLOCKS, num_sms());
  if (a.splits > 8 &&
      cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
    return check_cuda("cudaFuncSetAttribute(attn_decode cluster)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.splits, (unsigned)(a.Hk * groups), (unsigned)a.B);
  cfg.blockDim = dim3(F::THREADS);
  cfg.dynamicSmemBytes = F::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)a.splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tk, tv, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(PKM_ERR_CUDA, std::string("attn_decode_kernel launch: ") + cudaGetErrorString(e));
  }
  return PKM_OK;
}

template <typename T, int DP, bool Q4>
static int decode_rows(const DecodeArgs& a, const AttnArgs* dense, int64_t visible, cudaStream_t st) {
  return a.Tq * a.G > DC_ROWS ? decode_go<T, DP, 2, Q4>(a, dense, visible, st)
                              : decode_go<T, DP, 1, Q4>(a, dense, visible, st);
}

template <bool Q4>
static int decode_types(const DecodeArgs& a, const AttnArgs* dense, int64_t visible, int dtype, cudaStream_t st) {
  if (dtype == PKM_DT_BF16)
    return a.D > 64 ? decode_rows<__nv_bfloat16, 128, Q4>(a, dense, visible, st)
                    : decode_rows<__nv_bfloat16, 64, Q4>(a, dense, visible, st);
  return a.D > 64 ? decode_rows<__half, 128, Q4>(a, dense, visible, st)
                  : decode_rows<__half, 64, Q4>(a, dense, visible, st);
}

// Keys a row sees at most.
static int64_t visible_keys(int64_t rows, int64_t Tq, int64_t window, int64_t sinks) {
  return window ? std::min(rows, window + Tq - 1 + sinks) : rows;
}

int attn_decode_launch(const AttnArgs& f, int dtype, cudaStream_t st) {
  DecodeArgs a{};
  a.q = f.q;
  a.sq = f.sq;
  a.out = f.out;
  a.out_lo = f.out_lo;
  a.so = f.so;
  a.lse = f.lse;
  a.B = f.B;
  a.Hq = f.Hq;
  a.Hk = f.Hk;
  a.G = f.G;
  a.Tq = f.Tq;
  a.rows = f.Tk;
  a.D = f.D;
  a.scale = f.scale;
  a.window = f.window;
  a.sinks = f.sinks;
  a.starts = f.starts;
  a.ends = f.ends;
  a.err = f.err;
  return decode_types<false>(a, &f, visible_keys(f.Tk, f.Tq, f.window, f.sinks), dtype, st);
}

int kv4_attend_launch(const Kv4Attend& f, int dtype, cudaStream_t st) {
  DecodeArgs a{};
  a.q = f.q;
  a.sq = f.sq;
  a.out = f.out;
  a.so = f.so;
  for (int i = 0; i < 2; ++i) {
    a.codes[i] = f.codes[i];
    a.params[i] = f.params[i];
  }
  a.B = f.B;
  a.Hq = f.Hq;
  a.Hk = f.Hk;
  a.G = f.G;
  a.Tq = f.Tq;
  a.rows = f.cap;
  a.D = f.D;
  a.own_end = 1;
  a.scale = f.scale;
  a.window = f.window;
  a.sinks = f.sinks;
  a.starts = f.starts;
  a.ends = f.lengths;
  a.err = f.err;
  return decode_types<true>(a, nullptr, visible_keys(f.cap, f.Tq, f.window, f.sinks), dtype, st);
}

}  // namespace pkm
