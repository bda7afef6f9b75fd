// Decode attention over the 8-bit KV cache, with and without a prefix shared by the batch.
//
// Row (b, h) with keys j (the shared prefix's first, then the sequence's own):
//   z_j = (q . k_j) / sqrt(hd),  m = max_j z_j,  x_j = max(z_j - m, -87.3),
//   e_j = (12 + 6 x_j + x_j^2) / (12 - 6 x_j + x_j^2),  out = sum_j e_j v_j / sum_j e_j.
// e is the reference's rational FastExp (MathUtils.cs:20-32).  It is not multiplicative, so
// partial results against a running maximum cannot be rescaled: the exact maximum comes
// first and the weights are formed against it.
#include <cooperative_groups.h>

#include <algorithm>
#include <mutex>

#include "kv8.cuh"
#include "kv8_mma.cuh"
#include "mbar.cuh"

namespace sm {
namespace {

// ---------------------------------------------------------------- pieces of the decode kernels
//
// Keys are taken in blocks of 32, a warp each:
//   scores  two 16-key x 8-head MMA tiles.  K codes are A fragments as they lie: a lane takes 16
//           neighbouring bytes of a row, and q's digits, built once, are in the matching order.  A lane's
//           four rows are the keys whose scores the P side wants side by side.  Scores are kept as they are
//           compared and subtracted, so that x is 0 at the largest one, not a rounding above it;
//   P V     weights e, and P = e * v_scale in 23-bit fixed point against the largest v_scale of
//           the warp's keys, in the registers that the MMA wants them in; V codes are made
//           fragments by 4 x 4 byte transposes.  With up to 4 heads the three digits of all of
//           them are rows of one A operand; with more, a digit is a B operand of 8 heads.
// The kernels come with W = 8 and with W = 4 warps a CTA: the smaller CTAs, twice as many on an SM, hide one
// another's phases better once there are waves of them.
template <int HD, int GP>
struct Tile {
  static constexpr bool PA = GP == 4;           // P's digits as the A operand
  static constexpr int NT = GP > 8 ? 2 : 1;     // column tiles of 8 heads
  static constexpr int CP = GP > 8 ? 8 : GP;    // heads a tile keeps
  static constexpr int ZB = 32 * CP;            // scores of a block and column tile
  static constexpr int DS = HD == 128 && GP == 16 ? 2 : 1;  // warps that split the dims of a key block
  static constexpr int DP = HD / DS;            // dims a warp
  static constexpr int VB = DP / 8;             // bytes of a V row a lane
  // accumulator tiles: PA one for each byte of a lane (8 dims), else 16 dims x (heads, digits)
  static constexpr int MT = PA ? VB : DP / 16;
  static constexpr int MD = PA ? 1 : 3 * NT;
};

// Scores of a block lie as [head][t][8]: the scores of keys t + 4 i, i = 0..7, in a row.
// A lane's rows of the score tiles are keys krow(g) + 4 c, c = 0..3: half of such a row.
__device__ __forceinline__ int krow(int g) { return (g & 3) + 16 * (g >> 2); }
__device__ __forceinline__ int zpos(int head, int g) { return head * 32 + (g & 3) * 8 + (g >> 2) * 4; }

// q of one kv head's group as digits in B-fragment order; `unit` gets 2^e / sqrt(HD) of this lane's
// column head (lane / 4), the factor of its digit sums (NaN where q is not finite).
template <int HD, int GP>
__device__ __forceinline__ void load_q(const float* q, bool vec, int G, int lane,
                                       uint32_t (&qd)[Tile<HD, GP>::NT][HD / 32][3][2],
                                       float (&unit)[Tile<HD, GP>::NT]) {
  using T = Tile<HD, GP>;
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) {
    const int h = nt * 8 + g;
    float x[HD / 4];
    float peak = 0.f;
    if (vec) {
#pragma unroll
      for (int i = 0; i < HD / 4; i += 4)
        *(float4*)(x + i) = h < G ? *(const float4*)(q + h * HD + (i / 16) * 64 + 16 * t + i % 16) : float4{};
    } else {
#pragma unroll
      for (int i = 0; i < HD / 4; ++i) x[i] = h < G ? q[h * HD + (i / 16) * 64 + 16 * t + i % 16] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) peak = max_nan(peak, fabsf(x[i]));
    peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
    const bool ok = peak < INFINITY;
    const int e = ok ? query_exp(peak) : 0;
    const Scale2 up(22 - e);
    unit[nt] = ok ? query_unit<HD>(e) : NAN;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float* xs = x + 8 * i + 4 * half;
        bytes3((uint32_t)__float2int_rn(up(xs[0])), (uint32_t)__float2int_rn(up(xs[1])),
               (uint32_t)__float2int_rn(up(xs[2])), (uint32_t)__float2int_rn(up(xs[3])), qd[nt][i][0][half],
               qd[nt][i][1][half], qd[nt][i][2][half]);
      }
  }
}

// K codes and scales of a block, as a lane holds them: rows krow(g) + 4 c, bytes 16 t .. of each 64.
template <int HD>
struct KBlock {
  uint32_t w[4][HD / 64][4];
  float s[4];
};

// Factors of columns 2t, 2t + 1, from the lanes whose column heads they are
template <int NT>
__device__ __forceinline__ void column_units(const float (&unit)[NT], int t, float (&of)[NT][2]) {
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 2; ++i) of[nt][i] = __shfl_sync(0xffffffffu, unit[nt], (2 * t + i) * 4);
}

// Scores of a block: to z ([NT] planes `plane` floats apart), and this lane's running maxima of columns 2t, 2t + 1,
// whose factors are `unit`.  The factors meet first: a sum of up to 2^14 times a large scale would leave fp32's range
// where the score does not.
template <int HD, int GP>
__device__ __forceinline__ void score_block(const KBlock<HD>& k,
                                            const uint32_t (&qd)[Tile<HD, GP>::NT][HD / 32][3][2],
                                            const float (&unit)[Tile<HD, GP>::NT][2], int g, int t, float* z,
                                            int64_t plane, float (&mx)[Tile<HD, GP>::NT][2]) {
  using T = Tile<HD, GP>;
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) {
    float s[4][2];  // key krow(g) + 4 c, column 2t + i
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      int d[3][4] = {};
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const uint32_t a0 = k.w[2 * m][i >> 1][2 * (i & 1)], a2 = k.w[2 * m][i >> 1][2 * (i & 1) + 1];
        const uint32_t a1 = k.w[2 * m + 1][i >> 1][2 * (i & 1)], a3 = k.w[2 * m + 1][i >> 1][2 * (i & 1) + 1];
        mma_s8u8(d[0], a0, a1, a2, a3, qd[nt][i][0][0], qd[nt][i][0][1]);
        mma_s8u8(d[1], a0, a1, a2, a3, qd[nt][i][1][0], qd[nt][i][1][1]);
        mma_s8s8(d[2], a0, a1, a2, a3, qd[nt][i][2][0], qd[nt][i][2][1]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        s[2 * m + (i >> 1)][i & 1] = join3_query(d[2][i], d[1][i], d[0][i]) * (k.s[2 * m + (i >> 1)] * unit[nt][i & 1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mx[nt][i] = fmaxf(mx[nt][i], fmaxf(fmaxf(s[0][i], s[1][i]), fmaxf(s[2][i], s[3][i])));
      if (2 * t < T::CP)
        *(float4*)(z + nt * plane + zpos(2 * t + i, g)) = make_float4(s[0][i], s[1][i], s[2][i], s[3][i]);
    }
  }
}

// Maxima of a warp's columns (lanes g of one t merged) into to[GP]
template <int HD, int GP>
__device__ __forceinline__ void warp_maxima(const float (&mx)[Tile<HD, GP>::NT][2], int g, int t, float* to) {
#pragma unroll
  for (int nt = 0; nt < Tile<HD, GP>::NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float m = mx[nt][c];
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      if (g == 0 && 2 * t < Tile<HD, GP>::CP) to[nt * 8 + 2 * t + c] = m;
    }
}

// V codes of a block: keys t + 4 i, VB dims of each; and the scale of key `lane` (0 past the end).
template <int HD, int GP>
struct VBlock {
  uint32_t w[8][Tile<HD, GP>::VB / 4];
  float s;
};

// What a warp accumulates of P V, and how P is formed.
template <int HD, int GP>
struct PVSum {
  using T = Tile<HD, GP>;
  // A lane's head is column g of each tile and its keys are t + 4 i, i = 0..7.  With P as A, lanes g and
  // g + 4 share head g & 3: the first takes i = 0..3, the second i = 4..7.
  static constexpr int NZ = T::PA ? 4 : 8;
  static __device__ __forceinline__ int column(int g) { return T::PA ? g & 3 : g; }
  // where the lane's scores of a block and tile begin
  static __device__ __forceinline__ int zstart(int g, int t) {
    return T::PA ? (g & 3) * 32 + t * 8 + (g >> 2) * 4 : g * 32 + t * 8;
  }

  float m[T::NT], esum[T::NT];  // of this lane's head: maximum and sum of weights
  float top, inv;               // largest V scale and 1 / it
  int acc[T::MD][T::MT][4];

  // Fixed point: e = 1 at the largest scale is POINT = 2^23 - 8.  In two factors each way, so that none of them
  // leaves the normal numbers; scales below those keep their resolution.
  static constexpr float POINT = 8388600.f;
  __device__ __forceinline__ float value(float sum) const { return sum * (1.f / POINT) * top; }
  __device__ __forceinline__ void start(float vmax, const float (&max_of)[T::NT]) {
    top = max_nan(vmax, 0x1p-126f);
    inv = 1.f / top;
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) m[nt] = max_of[nt], esum[nt] = 0.f;
#pragma unroll
    for (int i = 0; i < T::MD; ++i)
#pragma unroll
      for (int c = 0; c < T::MT; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][c][e] = 0;
  }

  // zv: the lane's scores of each tile; keys: how many of the block's 32 exist.  v is used up.
  __device__ __forceinline__ void add(VBlock<HD, GP>& v, const float (&zv)[T::NT][NZ], int keys, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const int first = T::PA ? t + (g >> 2) * 16 : t;
    const float vsm = v.s * inv * POINT;
    uint32_t dg[T::NT][3][NZ / 4];
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) {
      float e[NZ];
#pragma unroll
      for (int i = 0; i < NZ; ++i) e[i] = kv8_weight(zv[nt][i] - m[nt]);
      if (keys < 32) {
#pragma unroll
        for (int i = 0; i < NZ; ++i)
          if (first + 4 * i >= keys) e[i] = 0.f;
      }
      float part = 0.f;
      uint32_t p[NZ];
#pragma unroll
      for (int i = 0; i < NZ; ++i) {
        part += e[i];
        // x <= 0, so e * scale lies in [0, 2^23): added to 2^23 it is the mantissa, rounded
        p[i] = __float_as_uint(fmaf(e[i], __shfl_sync(0xffffffffu, vsm, first + 4 * i), 8388608.f));
      }
      esum[nt] += part;
#pragma unroll
      for (int half = 0; half < NZ / 4; ++half)
        bytes3(p[4 * half], p[4 * half + 1], p[4 * half + 2], p[4 * half + 3], dg[nt][0][half], dg[nt][1][half],
               dg[nt][2][half]);
    }
#pragma unroll
    for (int c = 0; c < T::VB / 4; ++c) {
      transpose4(v.w[0][c], v.w[1][c], v.w[2][c], v.w[3][c]);
      transpose4(v.w[4][c], v.w[5][c], v.w[6][c], v.w[7][c]);
    }
    if constexpr (T::PA) {
      // rows: digit 0 of heads 0..3, digit 1, digit 2, zeros; lanes g and g + 4 exchange what the other's rows need
      const bool low = g < 4;
      const uint32_t x = __shfl_xor_sync(0xffffffffu, low ? dg[0][1][0] : dg[0][0][0], 16);
      const uint32_t y = __shfl_xor_sync(0xffffffffu, dg[0][2][0], 16);
      const uint32_t a0 = low ? dg[0][0][0] : x, a2 = low ? x : dg[0][1][0];
      const uint32_t a1 = low ? dg[0][2][0] : 0u, a3 = low ? y : 0u;
#pragma unroll
      for (int c = 0; c < T::MT; ++c)
        mma_u8s8_acc(acc[0][c], a0, a1, a2, a3, v.w[c & 3][c >> 2], v.w[4 + (c & 3)][c >> 2]);
    } else {
#pragma unroll
      for (int mt = 0; mt < T::MT; ++mt) {
        // the lane's bytes 2 mt and 2 mt + 1 are rows g and g + 8 of the tile
        const int c = mt >> 1, o = (mt & 1) * 2;
#pragma unroll
        for (int i = 0; i < 3 * T::NT; ++i)
          mma_s8u8(acc[i][mt], v.w[o][c], v.w[o + 1][c], v.w[4 + o][c], v.w[4 + o + 1][c], dg[i / 3][i % 3][0],
                   dg[i / 3][i % 3][1]);
      }
    }
  }

  // The warp's sums to to[GP][HD], its weights' to sums[GP] (of the warps at d0 == 0).
  __device__ __forceinline__ void store(float* to, float* sums, int lane, int d0) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) {
      esum[nt] += __shfl_xor_sync(0xffffffffu, esum[nt], 1);
      esum[nt] += __shfl_xor_sync(0xffffffffu, esum[nt], 2);
      if (T::PA) esum[nt] += __shfl_xor_sync(0xffffffffu, esum[nt], 16);
      if (t == 0 && g < T::CP && d0 == 0) sums[nt * 8 + g] = esum[nt];
    }
    if constexpr (T::PA) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float o[T::MT];
#pragma unroll
        for (int c = 0; c < T::MT; ++c)
          o[c] = value(join3(acc[0][c][2 + i], __shfl_xor_sync(0xffffffffu, acc[0][c][i], 16), acc[0][c][i]));
        if (g < 4) {
#pragma unroll
          for (int c = 0; c < T::MT; c += 4)
            *(float4*)(to + g * HD + (2 * t + i) * T::VB + c) = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
        }
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < T::MT; ++mt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float* p = to + (nt * 8 + 2 * t + i) * HD + d0 + g * T::VB + 2 * mt;
            *(float2*)p = make_float2(
                value(join3(acc[3 * nt + 2][mt][i], acc[3 * nt + 1][mt][i], acc[3 * nt][mt][i])),
                value(join3(acc[3 * nt + 2][mt][i + 2], acc[3 * nt + 1][mt][i + 2], acc[3 * nt][mt][i + 2])));
          }
    }
  }
};

// ---------------------------------------------------------------- a warp's ring
//
// Each warp streams its blocks through a ring of its own: asynchronous copies, some blocks ahead of the
// one it works on, and no barrier but the warp's.
//
// 16-byte chunk c of row r of a block sits at c ^ swizzle(r): with it neither the K side (lanes of two
// rows and 64 bytes at once) nor the V side (four rows, 32 bytes) meets a bank twice.
template <int HD>
__device__ __forceinline__ int swizzle(int r) {
  return HD == 128 ? ((r & 1) << 2) | (r & 2) : r & 2;
}

// One slot: codes of 32 rows, their V scales, then 128 bytes of K scales or (Z) the block's scores.
template <int HD, int GP, bool Z>
struct Slot {
  using T = Tile<HD, GP>;
  static constexpr int CODES = 32 * HD;
  static constexpr int MORE = CODES + 128;
  static constexpr int BYTES = MORE + (Z ? T::NT * T::ZB * 4 : 128);

  // rows at or past n repeat row n - 1; ks nullptr: none
  static __device__ __forceinline__ void fetch(uint32_t to, const int8_t* codes, const float* ks, const float* vs,
                                               int row, int n, int lane, uint64_t policy) {
    constexpr int C = HD / 16, R = 32 / C;  // chunks of a row; rows of 32 chunks
    const int r = lane / C;
    const uint32_t dst = to + r * HD + (((lane % C) ^ swizzle<HD>(r)) << 4);
    const int8_t* src = codes + (int64_t)(row + r) * HD + (lane % C) * 16;
    if (row + 32 <= n) {
#pragma unroll
      for (int j = 0; j < C; ++j) cp16(dst + j * 512, src + j * 512, policy);
    } else {
#pragma unroll
      for (int j = 0; j < C; ++j) cp16(dst + j * 512, src + min(j * R, n - 1 - row - r) * HD, policy);
    }
    const int s = min(row + lane, n - 1);
    cp4(to + CODES + 4 * lane, vs + s);
    if (ks) cp4(to + MORE + 4 * lane, ks + s);
  }
  // the block's scores, planes `plane` floats apart
  static __device__ __forceinline__ void fetch_scores(uint32_t to, const float* z, int64_t plane, int row, int lane) {
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
      for (int j = 0; j < T::ZB / 128; ++j)
        cp16(to + MORE + (nt * T::ZB + j * 128 + lane * 4) * 4,
             z + nt * plane + (int64_t)(row >> 5) * T::ZB + j * 128 + lane * 4);
  }
  static __device__ __forceinline__ void read_k(const uint8_t* p, KBlock<HD>& k, float& vmax, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int r = krow(g) + 4 * c;
#pragma unroll
      for (int l = 0; l < HD / 64; ++l)
        *(uint4*)k.w[c][l] = *(const uint4*)(p + r * HD + (((l * 4 + t) ^ swizzle<HD>(g)) << 4));
      k.s[c] = *(const float*)(p + MORE + 4 * r);
    }
    vmax = max_nan(vmax, *(const float*)(p + CODES + 4 * lane));
  }
  // keys: how many of the block's rows exist
  static __device__ __forceinline__ void read_v(const uint8_t* p, VBlock<HD, GP>& v, int keys, int d0, int lane) {
    const int g = lane >> 2, t = lane & 3, byte = d0 + g * T::VB;
    v.s = lane < keys ? *(const float*)(p + CODES + 4 * lane) : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint8_t* r = p + (t + 4 * i) * HD + (((byte >> 4) ^ swizzle<HD>(t)) << 4) + (byte & 15);
      if constexpr (T::VB == 16)
        *(uint4*)v.w[i] = *(const uint4*)r;
      else
        *(uint2*)v.w[i] = *(const uint2*)r;
    }
  }
};

// Largest of a warp's values, NaN if any is
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// ---------------------------------------------------------------- decode, short: one cluster per (sequence, kv head)
//
// One launch: the keys (a shared prefix's blocks first, then the sequence's own) are split over the cluster's
// CTAs, the scores stay in shared memory, and the exact maximum and the sums travel through distributed shared
// memory.  Behind a prefix (o) the weights are formed against the larger of both maxima and the sums are left to
// be joined.  A warp's K blocks and then its V blocks go through one ring, so V is on its way while the maxima
// are exchanged.  Bound by its chain of phases.
// CTAs of W warps an SM: what a group's accumulators leave registers for
template <int HD, int GP>
constexpr int ctas_by_registers(int W) {
  return (GP == 4 || (HD == 64 && GP == 8) ? 16 : 8) / W;
}

template <int HD, int GP, int W>
struct ClusterSmem {
  using T = Tile<HD, GP>;
  using S = Slot<HD, GP, false>;
  static constexpr int N = HD == 64 ? 4 : 3;     // ring slots
  static constexpr int RING = W * N * S::BYTES;
  static constexpr int TAIL = GP * HD + 2 * GP;  // this CTA's sums, maxima and weights for the cluster
  static_assert(RING >= W / T::DS * GP * HD * 4, "the warps' sums take the rings' place");
  static size_t bytes(int64_t cap) { return RING + ((size_t)cap * GP + TAIL) * sizeof(float); }
};

template <int HD, int GP, int W>
__global__ void __launch_bounds__(32 * W, ctas_by_registers<HD, GP>(W))
    decode_kv8_kernel(Kv8Attn a, Kv8Behind o, int cap) {
  using T = Tile<HD, GP>;
  using M = ClusterSmem<HD, GP, W>;
  constexpr int DW = W, DT = 32 * W, TW = W / T::DS;
  using S = Slot<HD, GP, false>;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), CL = (int)cluster.num_blocks();
  const int gk = blockIdx.y, b = blockIdx.z;
  const int G = a.n_heads / a.c.n_kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  extern __shared__ __align__(128) uint8_t smem[];
  float* z = (float*)(smem + M::RING);   // [NT][cap / 32] score blocks
  float* pacc = z + (int64_t)cap * GP;   // [GP][HD] this CTA's sums
  float* stat = pacc + GP * HD;          // [GP] maximum, [GP] sum of weights
  __shared__ float wred[DW][GP], vred[DW], gmax[GP];
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  int slot, len;
  if (!row_keys(a, b, slot, len)) return;
  float* out = a.out + ((int64_t)b * a.n_heads + gk * G) * HD;
  const int64_t row0 = (int64_t)gk * o.rows + (int64_t)b * G;  // behind a prefix
  if (a.prefix_len + len == 0) {
    if (rank == 0) {
      for (int i = tid; i < G * HD; i += DT) (o.prefix_max ? o.acc + row0 * HD : out)[i] = 0.f;
      if (o.prefix_max && tid < G) o.sum[row0 + tid] = 0.f;
    }
    return;
  }
  // this CTA's blocks of all: the prefix's np, then the sequence's own
  const int np = (a.prefix_len + 31) >> 5, all = np + ((len + 31) >> 5);
  const int per = (all + CL - 1) / CL;
  const int b0 = min(all, rank * per), blocks = min(all - b0, per);
  const int64_t own0 = a.c.at(slot, gk, 0), prefix0 = a.prefix.at(a.prefix_seq, gk, 0);
  const int64_t plane = (int64_t)cap * T::CP;
  // keys of a block
  auto keys_of = [&](int blk) {
    const int i = b0 + blk;
    return i < np ? a.prefix_len - 32 * i : len - 32 * (i - np);
  };
  // the warp's blocks: K blocks warp, warp + DW, ..; then V blocks tw, tw + TW, ..
  const int tw = warp / T::DS, d0 = (warp % T::DS) * T::DP;
  const int nk = (blocks - warp + DW - 1) / DW, nv = (blocks - tw + TW - 1) / TW;
  const uint8_t* ring = smem + warp * M::N * S::BYTES;
  const uint32_t ring_at = smem_u32(ring);
  const uint64_t once = l2_evict_first_policy(), often = l2_evict_normal_policy();
  auto fetch = [&](int i) {
    if (i < nk + nv) {
      const bool is_k = i < nk;
      const int blk = b0 + (is_k ? warp + DW * i : tw + TW * (i - nk));
      const bool shared = blk < np;
      const Kv8View& c = shared ? a.prefix : a.c;
      const int64_t at = shared ? prefix0 : own0;
      S::fetch(ring_at + i % M::N * S::BYTES, (is_k ? c.k : c.v) + at * HD, is_k ? c.ks + at : nullptr, c.vs + at,
               32 * (shared ? blk : blk - np), shared ? a.prefix_len : len, lane, shared ? often : once);
    }
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < M::N - 1; ++i) fetch(i);

  float vmax = 0.f;
  uint32_t qd[T::NT][HD / 32][3][2];
  float unit[T::NT], units[T::NT][2], mx[T::NT][2];
  load_q<HD, GP>(a.q + (int64_t)b * a.q_stride + (int64_t)gk * G * HD, a.q_vec, G, lane, qd, unit);
  column_units(unit, t, units);
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
  for (int i = 0; i < nk; ++i) {
    cp_wait<M::N - 2>();
    KBlock<HD> k;
    S::read_k(ring + i % M::N * S::BYTES, k, vmax, lane);
    fetch(i + M::N - 1);  // into the slot of block i - 1
    score_block<HD, GP>(k, qd, units, g, t, z + (warp + DW * i) * T::ZB, plane, mx);
  }
  warp_maxima<HD, GP>(mx, g, t, wred[warp]);
  vmax = warp_max_nan(vmax);
  if (lane == 0) vred[warp] = vmax;
  __syncthreads();
  float m = -INFINITY;
  if (tid < GP) {
#pragma unroll
    for (int i = 0; i < DW; ++i) m = fmaxf(m, wred[i][tid]);
    stat[tid] = m;
  }
#pragma unroll
  for (int i = 0; i < DW; ++i) vmax = max_nan(vmax, vred[i]);
  if (CL > 1) {
    cluster.sync();
    if (tid < GP)
      for (int r = 0; r < CL; ++r) m = fmaxf(m, cluster.map_shared_rank(stat, r)[tid]);
  }
  if (tid < GP) gmax[tid] = m;
  __syncthreads();

  PVSum<HD, GP> pv;
  const int col = pv.column(g);
  float max_of[T::NT];
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) {
    max_of[nt] = gmax[nt * 8 + col];
    const int h = nt * 8 + col;
    if (o.prefix_max && h < G) {
      if (rank == 0 && warp == 0 && t == 0 && g == col) o.own_max[row0 + h] = max_of[nt];
      max_of[nt] = fmaxf(max_of[nt], o.prefix_max[row0 + h]);
    }
  }
  pv.start(vmax, max_of);
  for (int i = nk; i < nk + nv; ++i) {
    const int blk = tw + TW * (i - nk);
    cp_wait<M::N - 2>();
    VBlock<HD, GP> v;
    S::read_v(ring + i % M::N * S::BYTES, v, keys_of(blk), d0, lane);
    fetch(i + M::N - 1);
    float zv[T::NT][pv.NZ];
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
      for (int c = 0; c < pv.NZ; c += 4)
        *(float4*)&zv[nt][c] = *(const float4*)(z + nt * plane + blk * T::ZB + pv.zstart(g, t) + c);
    pv.add(v, zv, keys_of(blk), lane);
  }
  cp_wait<0>();
  __syncthreads();  // the rings are done
  float* part = (float*)smem;  // [TW][GP][HD]
  pv.store(part + tw * GP * HD, wred[tw], lane, d0);
  __syncthreads();
  auto write = [&](int i, float s, float total) {
    if (o.prefix_max) {
      o.acc[row0 * HD + i] = s;
      if (i % HD == 0) o.sum[row0 + i / HD] = total;
    } else {
      out[i] = __fdiv_rn(s, total);
    }
  };
  for (int i = tid; i < G * HD; i += DT) {
    float s = 0.f, total = 0.f;
#pragma unroll
    for (int r = 0; r < TW; ++r) s += part[r * GP * HD + i], total += wred[r][i / HD];
    if (CL == 1) {
      write(i, s, total);
    } else {
      pacc[i] = s;
      if (i % HD == 0) stat[GP + i / HD] = total;
    }
  }
  if (CL == 1) return;
  cluster.sync();
  // each rank its share of the outputs
  for (int i = rank * DT + tid; i < G * HD; i += CL * DT) {
    float s = 0.f, total = 0.f;
    for (int r = 0; r < CL; ++r) {
      s += cluster.map_shared_rank(pacc, r)[i];
      total += cluster.map_shared_rank(stat, r)[GP + i / HD];
    }
    write(i, s, total);
  }
  cluster.sync();  // no CTA's shared memory goes before the others have read it
}

// ---------------------------------------------------------------- decode, long: scores, then P V, as two launches
//
// Flat grids over chunks of keys, so that nothing waits inside a kernel: the scores of a chunk go to
// global memory with the chunk's maxima (and its largest V scale), the second kernel reads them back
// against the maximum over the chunks; the CTA that finishes a (sequence, kv head) joins its chunks'
// sums, in order.  The scores add GP * 8 bytes to the 2 * HD + 8 of a key and mostly stay in L2.  Bound by
// HBM.
struct Kv8Split {
  Kv8Attn a;
  Kv8Behind o;
  int chunk, n_chunks;  // keys of a chunk (whole blocks); chunks that max_len makes
  int gp;               // heads a kv head's group is padded to: 4, 8 or 16
  int warps;            // of a CTA: 4 or 8
  float* z;             // [B][n_kv][gp / 8 or 1][blocks] blocks of scores
  float* pacc;          // [B][n_kv][n_chunks][gp][head_dim]
  float* stat;          // [B][n_kv][n_chunks][2 * gp + 1] maxima, largest V scale; then the weights' sums
  int* arrived;         // [B][n_kv] chunks whose P V is done
};

template <int HD, int GP, int W, bool PV>
struct SplitSmem {
  using S = Slot<HD, GP, PV>;
  static constexpr int CTAS = PV ? ctas_by_registers<HD, GP>(W) : (GP == 16 ? 8 : 16) / W;
  // as many slots as the CTAs of an SM have room for
  static constexpr int FIT = 224 / CTAS * 1024 / (W * S::BYTES);
  static constexpr int N = FIT > 6 ? 6 : FIT;
  static constexpr int RING = W * N * S::BYTES;
  static_assert(N >= 3 && RING >= W / Tile<HD, GP>::DS * GP * HD * 4, "ring too small");
};

template <int HD, int GP, int W>
__global__ void __launch_bounds__(32 * W, (SplitSmem<HD, GP, W, false>::CTAS)) split_scores_kernel(Kv8Split s) {
  using T = Tile<HD, GP>;
  using S = Slot<HD, GP, false>;
  using M = SplitSmem<HD, GP, W, false>;
  constexpr int DW = W;
  const Kv8Attn& a = s.a;
  const int ch = blockIdx.x, gk = blockIdx.y, b = blockIdx.z;
  const int G = a.n_heads / a.c.n_kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float wred[DW][GP], vred[DW];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  // only now: what the next kernel reads before its own wait has then been written
  asm volatile("griddepcontrol.launch_dependents;");
  int slot, len;
  if (!row_keys(a, b, slot, len)) return;
  const int j0 = ch * s.chunk, n = min(len - j0, s.chunk);
  if (ch == 0 && tid == 0) s.arrived[(int64_t)b * a.c.n_kv + gk] = 0;
  if (n <= 0) return;
  const int64_t row0 = a.c.at(slot, gk, j0);
  const int8_t* kp = a.c.k + row0 * HD;
  const float* ksp = a.c.ks + row0;
  const float* vsp = a.c.vs + row0;
  const int64_t bg = (int64_t)b * a.c.n_kv + gk;
  const int64_t plane = (int64_t)s.n_chunks * s.chunk * T::CP;
  float* z = s.z + bg * T::NT * plane + (int64_t)(j0 >> 5) * T::ZB;
  const uint8_t* ring = smem + warp * M::N * S::BYTES;
  const uint32_t ring_at = smem_u32(ring);
  const uint64_t policy = l2_evict_first_policy();
  // block i of the warp starts at row 32 (warp + DW i), slot i % N
  auto fetch = [&](int row, int at) {
    if (row < n) S::fetch(ring_at + at * S::BYTES, kp, ksp, vsp, row, n, lane, policy);
    cp_commit();
  };
#pragma unroll
  for (int i = 0; i < M::N - 1; ++i) fetch(32 * (warp + DW * i), i);
  float vmax = 0.f;
  uint32_t qd[T::NT][HD / 32][3][2];
  float unit[T::NT], units[T::NT][2], mx[T::NT][2];
  load_q<HD, GP>(a.q + (int64_t)b * a.q_stride + (int64_t)gk * G * HD, a.q_vec, G, lane, qd, unit);
  column_units(unit, t, units);
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) mx[nt][0] = mx[nt][1] = -INFINITY;
  int at = 0;
  for (int row = 32 * warp; row < n; row += 32 * DW) {
    cp_wait<M::N - 2>();
    KBlock<HD> k;
    S::read_k(ring + at * S::BYTES, k, vmax, lane);
    // the slot of the block before this one is free
    fetch(row + 32 * DW * (M::N - 1), at == 0 ? M::N - 1 : at - 1);
    at = at == M::N - 1 ? 0 : at + 1;
    score_block<HD, GP>(k, qd, units, g, t, z + (int64_t)(row >> 5) * T::ZB, plane, mx);
  }
  cp_wait<0>();
  warp_maxima<HD, GP>(mx, g, t, wred[warp]);
  vmax = warp_max_nan(vmax);
  if (lane == 0) vred[warp] = vmax;
  __syncthreads();
  float* stat = s.stat + (bg * s.n_chunks + ch) * (2 * GP + 1);
  if (tid < GP) {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < DW; ++i) m = fmaxf(m, wred[i][tid]);
    stat[tid] = m;
    if (s.o.prefix_max && tid < G)
      atomic_max(s.o.own_max + (int64_t)gk * s.o.rows + (int64_t)b * G + tid, m);
  } else if (tid == GP) {
#pragma unroll
    for (int i = 0; i < DW; ++i) vmax = max_nan(vmax, vred[i]);
    stat[GP] = vmax;
  }
}

template <int HD, int GP, int W>
__global__ void __launch_bounds__(32 * W, (SplitSmem<HD, GP, W, true>::CTAS)) split_pv_kernel(Kv8Split s) {
  using T = Tile<HD, GP>;
  using S = Slot<HD, GP, true>;
  using M = SplitSmem<HD, GP, W, true>;
  constexpr int DW = W, DT = 32 * W, TW = W / T::DS;
  const Kv8Attn& a = s.a;
  const int ch = blockIdx.x, gk = blockIdx.y, b = blockIdx.z;
  const int G = a.n_heads / a.c.n_kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float wred[DW][GP], gmax[DW][GP];
  __shared__ bool last;
  // everything but the scores and maxima was there before the first kernel let this one start; a CTA without work
  // waits too, or the grid could end before the one it depends on
  int slot, len;
  if (!row_keys(a, b, slot, len)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const int j0 = ch * s.chunk, n = min(len - j0, s.chunk);
  const int64_t row0 = (int64_t)gk * s.o.rows + (int64_t)b * G;  // behind a prefix
  if (n <= 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (len == 0 && ch == 0) {
      float* to = s.o.prefix_max ? s.o.acc + row0 * HD : a.out + ((int64_t)b * a.n_heads + gk * G) * HD;
      for (int i = tid; i < G * HD; i += DT) to[i] = 0.f;
      if (s.o.prefix_max && tid < G) s.o.sum[row0 + tid] = 0.f;
    }
    return;
  }
  const int64_t first = a.c.at(slot, gk, j0);
  const int8_t* vp = a.c.v + first * HD;
  const float* vsp = a.c.vs + first;
  const int64_t bg = (int64_t)b * a.c.n_kv + gk;
  const int64_t plane = (int64_t)s.n_chunks * s.chunk * T::CP;
  const int tw = warp / T::DS, d0 = (warp % T::DS) * T::DP;
  const float* z = s.z + bg * T::NT * plane + (int64_t)(j0 >> 5) * T::ZB;
  const uint8_t* ring = smem + warp * M::N * S::BYTES;
  const uint32_t ring_at = smem_u32(ring);
  const uint64_t policy = l2_evict_first_policy();
#pragma unroll
  for (int i = 0; i < M::N - 1; ++i)
    if (32 * (tw + TW * i) < n)
      S::fetch(ring_at + i * S::BYTES, vp, nullptr, vsp, 32 * (tw + TW * i), n, lane, policy);
  // the maximum over the sequence's chunks
  PVSum<HD, GP> pv;
  const int col = pv.column(g);
  float* stat = s.stat + bg * s.n_chunks * (2 * GP + 1);
  const int used = (len + s.chunk - 1) / s.chunk;
  float max_of[T::NT];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
#pragma unroll
  for (int i = 0; i < M::N - 1; ++i) {
    const int row = 32 * (tw + TW * i);
    if (row < n) S::fetch_scores(ring_at + i * S::BYTES, z, plane, row, lane);
    cp_commit();  // the first group holds all of the codes so far
  }
  if (lane < GP) {
    float m = -INFINITY;
    for (int i = warp; i < used; i += DW) m = fmaxf(m, stat[i * (2 * GP + 1) + lane]);
    gmax[warp][lane] = m;
  }
  const float vmax = stat[ch * (2 * GP + 1) + GP];
  __syncthreads();
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) {
    max_of[nt] = -INFINITY;
#pragma unroll
    for (int i = 0; i < DW; ++i) max_of[nt] = fmaxf(max_of[nt], gmax[i][nt * 8 + col]);
    if (s.o.prefix_max && nt * 8 + col < G) max_of[nt] = fmaxf(max_of[nt], s.o.prefix_max[row0 + nt * 8 + col]);
  }
  pv.start(vmax, max_of);
  int at = 0;
  for (int row = 32 * tw; row < n; row += 32 * TW) {
    cp_wait<M::N - 2>();
    const uint8_t* p = ring + at * S::BYTES;
    float zv[T::NT][pv.NZ];
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
      for (int i = 0; i < pv.NZ; i += 4)
        *(float4*)&zv[nt][i] = *((const float4*)(p + S::MORE) + (nt * T::ZB + pv.zstart(g, t) + i) / 4);
    VBlock<HD, GP> v;
    S::read_v(p, v, n - row, d0, lane);
    const int next = row + 32 * TW * (M::N - 1);
    if (next < n) {
      const uint32_t to = ring_at + (at == 0 ? M::N - 1 : at - 1) * S::BYTES;
      S::fetch(to, vp, nullptr, vsp, next, n, lane, policy);
      S::fetch_scores(to, z, plane, next, lane);
    }
    cp_commit();
    at = at == M::N - 1 ? 0 : at + 1;
    pv.add(v, zv, n - row, lane);
  }
  cp_wait<0>();
  __syncthreads();  // the rings are done
  float* part = (float*)smem;  // [TW][GP][HD]
  pv.store(part + tw * GP * HD, wred[tw], lane, d0);
  __syncthreads();
  float* pacc = s.pacc + (bg * s.n_chunks + ch) * GP * HD;
  for (int i = tid; i < G * HD; i += DT) {
    float x = 0.f;
#pragma unroll
    for (int r = 0; r < TW; ++r) x += part[r * GP * HD + i];
    pacc[i] = x;
  }
  if (tid < GP) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < TW; ++i) x += wred[i][tid];
    stat[ch * (2 * GP + 1) + GP + 1 + tid] = x;
  }
  // the last CTA of this (sequence, kv head) joins the chunks, always in their order
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(s.arrived + bg, 1) == used - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int i = tid; i < G * HD; i += DT) {
    float x = 0.f, total = 0.f;
#pragma unroll 8
    for (int c = 0; c < used; ++c) {
      x += __ldcg(s.pacc + (bg * s.n_chunks + c) * GP * HD + i);
      total += __ldcg(stat + c * (2 * GP + 1) + GP + 1 + i / HD);
    }
    if (s.o.prefix_max) {
      s.o.acc[row0 * HD + i] = x;
      if (i % HD == 0) s.o.sum[row0 + i / HD] = total;
    } else {
      a.out[((int64_t)b * a.n_heads + gk * G) * HD + i] = __fdiv_rn(x, total);
    }
  }
}

constexpr size_t SMEM_MAX = 220 * 1024;

// How the cluster form would run, or size 0 where its scores do not fit or the split form is faster.
//
// Size: CTAs of one cluster have to be resident together, and a second wave of clusters waits for whole
// groups of SMs, so the largest size is taken whose clusters are all resident at once (32 / 4 heads of 64,
// 16 rows of up to 1024 keys: 4 CTAs 7.7 us, 8 CTAs, which are not, 13.6 us), with 128 keys a CTA at least
// and none up to 512 keys (32 / 4 x 64, 8 rows: at 512 keys 1 CTA 5.8 us, 4 CTAs 6.8 us; at 2048 keys 1 CTA 12 us,
// 8 CTAs 7.7 us), nor 2 CTAs below 2048 keys of 128 dims (32 / 8 x 128, 16 rows of 1024: 1 CTA 10.3 us, 2 CTAs
// 12.1 us).
//
// 4 warps a CTA instead of 8 where there is more than one wave of them and three (with many heads two) fit an SM
// (b 256, at 256 keys: 32 / 8 x 128 38 us against 53 us, 32 / 4 x 64 13 us against 19 us; but b 64, which is less than
// a wave, 7.4 us against 6.2 us).
//
// Split above 600 KB of codes an SM that has a CTA: at 262 KB (32 / 4 x 64, b 1, 32768 keys) 14.7 us against 18.3 us
// split, at 1 MB (32 / 8 x 128, b 1, 32768 keys) 29 us against 23 us, at 2 MB (16 / 16 x 128, b 1, 32768 keys) 54 us
// against 29 us; but never where a sequence has at most 128 KB of codes a head, nor from 8 small CTAs an SM on, for
// the split form's second launch then costs more than its larger rings gain (32 / 8 x 128, b 64: at 512 keys the same,
// at 1024 keys 36 us against 29 us split; b 256: at 512 keys 55 us against 65 us, at 1024 keys 96 us against 109 us;
// 32 / 4 x 64, b 256: at 1024 keys 37 us against 44 us, at 1536 keys, where no three fit, 69 us against 56 us).
// Behind a shared prefix, which L2 holds, the other form is attn_kv8_tc.cu, whose five launches take 30 to 40 us at
// least where head_dim is 128: there the bound is 1056 KB (32 / 8 x 128, prefix of 4096: 16 rows, 1056 KB, 28 us
// against 40 us; prefix of 1024: 64 rows, 1024 KB, 32 us against 41 us; 32 / 4 x 64, prefix of 4096, 64 rows, 950 KB:
// 42 us against 32 us).  Beyond it neither is faster everywhere until 1.4 MB (32 / 8 x 128, 16 rows: 1109 KB 34 us
// against 55 us, 1356 KB 40 us against 45 us; 16 / 16 x 128, 16 rows over 3000: 1353 KB 44 us against 42 us; 12 / 4 x
// 128, 64 rows over 3000: 1353 KB 44 us against 38 us) and then the matrix form is (1827 KB 56 us against 45 us).
struct ClusterPlan {
  int size, cap, warps;
  size_t smem;
};

template <int HD, int GP>
int plan_cluster(const Kv8Attn& a, int B, int device, int sms, ClusterPlan& plan) {
  using M = ClusterSmem<HD, GP, 8>;
  auto kern = decode_kv8_kernel<HD, GP, 8>;
  // clusters of 1, 2, 4, 8, 16 CTAs resident at once, by CTAs of all the shared memory and of what fits twice
  static int resident[64][2][5] = {};
  static size_t twice[64] = {};
  static bool ready[64] = {};
  static std::mutex mu;
  if (device >= 64) return fail(SM_ERR_UNSUPPORTED, "attention_kv8: device id too large");
  std::lock_guard<std::mutex> lock(mu);
  if (!ready[device]) {
    SM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX));
    SM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaFuncAttributes fa;
    int per_sm = 0, reserved = 0;
    SM_CUDA_TRY(cudaFuncGetAttributes(&fa, kern));
    SM_CUDA_TRY(cudaDeviceGetAttribute(&per_sm, cudaDevAttrMaxSharedMemoryPerMultiprocessor, device));
    SM_CUDA_TRY(cudaDeviceGetAttribute(&reserved, cudaDevAttrReservedSharedMemoryPerBlock, device));
    twice[device] = (per_sm / 2 - reserved - fa.sharedSizeBytes) & ~(size_t)127;
    for (int half = 0; half < 2; ++half)
      for (int i = 0; i < 5; ++i) {
        cudaLaunchAttribute attr[2];
        const size_t smem = half ? twice[device] : SMEM_MAX;
        cudaLaunchConfig_t probe = launch_config(dim3(1 << i), 256, smem, nullptr, 1 << i, attr);
        int fit = 0;
        if (cudaOccupancyMaxActiveClusters(&fit, (const void*)kern, &probe) != cudaSuccess) {
          cudaGetLastError();
          fit = 0;
        }
        resident[device][half][i] = fit;
      }
    ready[device] = true;
  }
  const int64_t bg = (int64_t)B * a.c.n_kv;
  const int64_t blocks = ((int64_t)a.prefix_len + 31) / 32 + ((int64_t)a.max_len + 31) / 32, keys = 32 * blocks;
  constexpr int AN_SM = ctas_by_registers<HD, GP>(8);
  const size_t smem4 = ClusterSmem<HD, GP, 4>::bytes(keys);
  plan = {};
  for (int i = 4; i >= 0; --i) {
    const int cl = 1 << i;
    if (cl > 1 && (keys <= 512 || cl * 128 > keys)) continue;
    if (cl == 2 && HD == 128 && keys < 2048) continue;
    const int64_t cap = 32 * ((blocks + cl - 1) / cl);
    const size_t smem = M::bytes(cap);
    const int fit = resident[device][smem <= twice[device]][i];
    if (smem > SMEM_MAX || (cl > 1 && bg > fit)) continue;
    const int64_t codes = keys * 2 * HD, ctas = bg * cl;
    const int64_t most = a.prefix_len > 0 && HD == 128 ? 1056 * 1024 : 600 * 1024;
    const bool small = cl == 1 && bg > (int64_t)AN_SM * sms && smem4 <= (AN_SM == 2 ? 74 : 112) * 1024;
    const bool waves = small && bg >= 8ll * sms && a.prefix_len == 0;
    if (codes <= 128 * 1024 || bg * codes / (ctas < sms ? ctas : sms) <= most || waves)
      plan = {cl, (int)cap, small ? 4 : 8, small ? smem4 : smem};
    break;
  }
  return SM_OK;
}

template <int HD, int GP>
int launch_decode_cluster(const Kv8Attn& a, const Kv8Behind& o, int B, const ClusterPlan& plan, cudaStream_t st) {
  cudaLaunchAttribute attr[2];
  auto kern = plan.warps == 4 ? decode_kv8_kernel<HD, GP, 4> : decode_kv8_kernel<HD, GP, 8>;
  if (plan.warps == 4)
    SM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX));
  const cudaLaunchConfig_t cfg =
      launch_config(dim3(plan.size, a.c.n_kv, B), 32 * plan.warps, plan.smem, st, plan.size, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, o, plan.cap));
  return SM_OK;
}

template <int HD, int GP, int W>
int launch_split_kernel(const Kv8Split& s, int B, bool pv, cudaStream_t st) {
  auto kern = pv ? split_pv_kernel<HD, GP, W> : split_scores_kernel<HD, GP, W>;
  const int smem = pv ? SplitSmem<HD, GP, W, true>::RING : SplitSmem<HD, GP, W, false>::RING;
  SM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = launch_config(dim3(s.n_chunks, s.a.c.n_kv, B), 32 * W, smem, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, s));
  return SM_OK;
}

template <int W>
int launch_split_as(const Kv8Split& s, int hd, int B, bool pv, cudaStream_t st) {
  if (hd == 64)
    return s.gp == 4   ? launch_split_kernel<64, 4, W>(s, B, pv, st)
           : s.gp == 8 ? launch_split_kernel<64, 8, W>(s, B, pv, st)
                       : launch_split_kernel<64, 16, W>(s, B, pv, st);
  return s.gp == 4   ? launch_split_kernel<128, 4, W>(s, B, pv, st)
         : s.gp == 8 ? launch_split_kernel<128, 8, W>(s, B, pv, st)
                     : launch_split_kernel<128, 16, W>(s, B, pv, st);
}

// Sizes the split form and returns the floats that its arrays take together.
int64_t plan_split(Kv8Split& s, int hd, int B, int sms) {
  const int G = s.a.n_heads / s.a.c.n_kv;
  s.gp = G <= 4 ? 4 : G <= 8 ? 8 : 16;
  const int64_t bg = (int64_t)B * s.a.c.n_kv;
  // one wave of CTAs (2 an SM, or 1 where a group's accumulators fill the registers) where that makes chunks of
  // 512 to 4096 keys (b 1, 131071 keys, 32 / 8 x 128: chunks of 1024 keys 76 us, of 2048 62 us, one wave of
  // 3552 54 us; b 64, 4096 to 8192 keys: of 1024 193 us, of 2048 159 us, of 4096 154 us)
  const int ctas = s.gp == 4 || (hd == 64 && s.gp == 8) ? 2 : 1;
  const int64_t wave = std::max<int64_t>(1, (int64_t)ctas * sms / bg);
  // 4 warps a CTA where there are waves of single chunks (32 / 8 x 128: b 64, 1024 keys 29 us against 36 us, b 256, 512
  // to 2048 keys 128 us against 141 us; longer ones the same time, and few sequences 57 us against 54 us)
  s.warps = wave == 1 && s.a.max_len <= 4096 ? 4 : 8;
  s.chunk = (int)std::min<int64_t>(4096, std::max<int64_t>(512, ((s.a.max_len + wave - 1) / wave + 31) & ~31LL));
  s.n_chunks = ceil_div(s.a.max_len, s.chunk);
  const int64_t rows = bg * s.n_chunks;
  return rows * s.chunk * s.gp + rows * s.gp * hd + rows * (2 * s.gp + 1) + bg;
}

int launch_split(Kv8Split& s, float* base, int hd, int B, cudaStream_t st) {
  const int64_t rows = (int64_t)B * s.a.c.n_kv * s.n_chunks;
  s.z = base;
  s.pacc = s.z + rows * s.chunk * s.gp;
  s.stat = s.pacc + rows * s.gp * hd;
  s.arrived = (int*)(s.stat + rows * (2 * s.gp + 1));
  for (bool pv : {false, true})
    SM_TRY(s.warps == 4 ? launch_split_as<4>(s, hd, B, pv, st) : launch_split_as<8>(s, hd, B, pv, st));
  return SM_OK;
}

int launch_decode_split(const Kv8Attn& a, int hd, int B, int sms, cudaStream_t st) {
  Kv8Split s = {};
  s.a = a;
  void* buf = nullptr;
  if (cudaMallocAsync(&buf, (size_t)plan_split(s, hd, B, sms) * sizeof(float), st) != cudaSuccess) {
    cudaGetLastError();
    return fail(SM_ERR_OOM, "attention_kv8: device allocation failed");
  }
  const int rc = launch_split(s, (float*)buf, hd, B, st);
  cudaFreeAsync(buf, st);
  return rc;
}

template <int HD, int GP>
struct ClusterForm {
  static int plan(const Kv8Attn& a, int B, int device, int sms, ClusterPlan& p) {
    return plan_cluster<HD, GP>(a, B, device, sms, p);
  }
  static int launch(const Kv8Attn& a, const Kv8Behind& o, int B, const ClusterPlan& p, cudaStream_t st) {
    return launch_decode_cluster<HD, GP>(a, o, B, p, st);
  }
};

// f of the cluster form's instance for a head dim and group
template <typename F>
int with_cluster_form(int hd, int G, F f) {
  if (hd == 64) return G <= 4 ? f(ClusterForm<64, 4>()) : G <= 8 ? f(ClusterForm<64, 8>()) : f(ClusterForm<64, 16>());
  return G <= 4 ? f(ClusterForm<128, 4>()) : G <= 8 ? f(ClusterForm<128, 8>()) : f(ClusterForm<128, 16>());
}

int launch_decode(const Kv8Attn& a, int hd, int B, int device, int sms, cudaStream_t st, int* n_launch) {
  ClusterPlan plan;
  SM_TRY(with_cluster_form(hd, a.n_heads / a.c.n_kv, [&](auto form) {
    SM_TRY(form.plan(a, B, device, sms, plan));
    return plan.size ? form.launch(a, Kv8Behind{}, B, plan, st) : SM_OK;
  }));
  *n_launch = plan.size ? 1 : 0;
  if (plan.size) return SM_OK;
  if (a.prefix_len > 0) return launch_attention_shared_tc(a, hd, B, device, sms, st, n_launch);
  *n_launch = 2;
  return launch_decode_split(a, hd, B, sms, st);
}

int attend(sm_ctx* ctx, const Kv8Attn& args, int head_dim, int B, const char* what) {
  int device = 0;
  cudaStream_t st = nullptr;
  int64_t* launches = nullptr;
  SM_TRY(ctx_view(ctx, &device, &st, &launches));
  DeviceGuard guard(device);
  Kv8Attn a = args;
  a.status = ctx_status(ctx);
  if (B > 65535 || a.c.n_kv > 65535) return fail(SM_ERR_SHAPE, std::string(what) + ": batch too large");
  int sms = 0, nl = 0;
  SM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  SM_TRY(launch_decode(a, head_dim, B, device, sms, st, &nl));
  *launches += nl;
  return SM_OK;
}

bool q_rows_vec(const float* q, int64_t q_stride) { return (uintptr_t)q % 16 == 0 && q_stride % 4 == 0; }

int check_attn(sm_ctx* ctx, const sm_kv8* c, const float* q, int64_t q_stride, const int* seq_ids, const int* lens,
               int max_len, int B, int n_heads, const float* out, const char* what) {
  auto refuse = [&](int code, const char* why) { return fail(code, std::string(what) + ": " + why); };
  SM_TRY(kv8_check(c, what));
  if (B < 0 || n_heads <= 0 || n_heads % c->n_kv) return refuse(SM_ERR_SHAPE, "bad shape");
  if (n_heads / c->n_kv > 16) return refuse(SM_ERR_UNSUPPORTED, "more than 16 q heads per kv head");
  if (max_len < 0 || max_len > c->max_tokens) return refuse(SM_ERR_SHAPE, "max_len outside 0 .. max_tokens");
  if (q_stride < (int64_t)n_heads * c->head_dim) return refuse(SM_ERR_SHAPE, "q_stride is less than a row");
  if (!seq_ids && B > c->max_seqs) return refuse(SM_ERR_SHAPE, "more rows than slots");
  if (!ctx || (B && (!q || !lens || !out))) return refuse(SM_ERR_INVALID_ARG, "null argument");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)seq_ids | (uintptr_t)lens) % 4)
    return refuse(SM_ERR_INVALID_ARG, "misaligned pointer");
  return SM_OK;
}

}  // namespace

int plan_kv8_own(Kv8Own& own, int hd, int B, int device, int sms) {
  ClusterPlan plan;
  SM_TRY(with_cluster_form(hd, own.a.n_heads / own.a.c.n_kv,
                           [&](auto form) { return form.plan(own.a, B, device, sms, plan); }));
  own.cluster = plan.size;
  own.cap = plan.cap;
  own.warps = plan.warps;
  own.smem = plan.smem;
  Kv8Split s = {};
  s.a = own.a;
  own.floats = plan.size ? 0 : plan_split(s, hd, B, sms);
  return SM_OK;
}

int launch_kv8_own(const Kv8Own& own, float* workspace, int hd, int B, int sms, cudaStream_t st, int* n_launch) {
  if (own.cluster) {
    ++*n_launch;
    return with_cluster_form(hd, own.a.n_heads / own.a.c.n_kv, [&](auto form) {
      return form.launch(own.a, own.behind, B, ClusterPlan{own.cluster, own.cap, own.warps, own.smem}, st);
    });
  }
  *n_launch += 2;
  Kv8Split s = {};
  s.a = own.a;
  s.o = own.behind;
  plan_split(s, hd, B, sms);
  return launch_split(s, workspace, hd, B, st);
}

}  // namespace sm

using namespace sm;

extern "C" {

SM_API int sm_attention_decode_kv8(sm_ctx* ctx, const sm_kv8* cache, const float* q, int64_t q_stride,
                                   const int* seq_ids, const int* lens, int max_len, int B, int n_heads,
                                   float* out) {
  const char* what = "attention_decode_kv8";
  SM_TRY(check_attn(ctx, cache, q, q_stride, seq_ids, lens, max_len, B, n_heads, out, what));
  if (B == 0) return SM_OK;
  Kv8Attn a{kv8_view(cache), {}, 0, 0, q, q_stride, seq_ids, lens, max_len, n_heads,
            out, nullptr, q_rows_vec(q, q_stride)};
  return attend(ctx, a, cache->head_dim, B, what);
}

SM_API int sm_attention_shared_kv8(sm_ctx* ctx, const sm_kv8* prefix, int prefix_seq, int prefix_len,
                                   const sm_kv8* cache, const float* q, int64_t q_stride, const int* seq_ids,
                                   const int* lens, int max_len, int B, int n_heads, float* out) {
  const char* what = "attention_shared_kv8";
  SM_TRY(kv8_check(cache, what));
  SM_TRY(kv8_check(prefix, what));
  if (prefix->n_kv != cache->n_kv || prefix->head_dim != cache->head_dim)
    return fail(SM_ERR_SHAPE, std::string(what) + ": the two caches' heads differ");
  if (prefix_seq < 0 || prefix_seq >= prefix->max_seqs || prefix_len < 0 || prefix_len > prefix->max_tokens)
    return fail(SM_ERR_SHAPE, std::string(what) + ": prefix outside its cache");
  if ((int64_t)prefix_len + max_len > INT32_MAX)
    return fail(SM_ERR_SHAPE, std::string(what) + ": context too long");
  SM_TRY(check_attn(ctx, cache, q, q_stride, seq_ids, lens, max_len, B, n_heads, out, what));
  if (B == 0) return SM_OK;
  Kv8Attn a{kv8_view(cache), kv8_view(prefix), prefix_seq, prefix_len, q, q_stride, seq_ids, lens, max_len, n_heads,
            out, nullptr, q_rows_vec(q, q_stride)};
  return attend(ctx, a, cache->head_dim, B, what);
}

}  // extern "C"
