// Decode attention over the 8-bit KV cache, with and without a prefix shared by the batch.
//
// Row (b, h) with keys j (the shared prefix's first, then the sequence's own):
//   z_j = (q . k_j) / sqrt(hd),  m = max_j z_j,  x_j = max(z_j - m, -87.3),
//   e_j = (12 + 6 x_j + x_j^2) / (12 - 6 x_j + x_j^2),  out = sum_j e_j v_j / sum_j e_j.
// e is the reference's rational FastExp (MathUtils.cs:20-32).  It is not multiplicative, so
// partial results against a running maximum cannot be rescaled: the exact maximum comes
// first and the weights are formed against it.
#include <cooperative_groups.h>

#include "kv8.cuh"
#include "kv8_mma.cuh"

namespace sm {
namespace {

struct Kv8Attn {
  Kv8View c, prefix;  // prefix.k == nullptr: none
  int prefix_seq, prefix_len;
  const float* q;
  int64_t q_stride;
  const int* seq_ids;
  const int* lens;
  int max_len, n_heads;
  float* out;
  int* status;
};

constexpr int THREADS = 128;

// One CTA per (query head, sequence): the scores are formed twice, a key a thread.
template <int HD>
__global__ void __launch_bounds__(THREADS) attn_kv8_kernel(Kv8Attn a) {
  const int h = blockIdx.x, b = blockIdx.y;
  const int g = h / (a.n_heads / a.c.n_kv);
  const int slot = a.seq_ids ? a.seq_ids[b] : b;
  if (slot < 0) return;
  const int len = a.lens[b];
  if (slot >= a.c.slots || len < 0 || len > a.max_len) {
    if (threadIdx.x == 0) atomicExch(a.status, SM_ERR_SHAPE);
    return;
  }
  __shared__ float qs[HD], es[THREADS], red[THREADS / 32];
  const float scale = 1.f / sqrtf((float)HD);
  for (int d = threadIdx.x; d < HD; d += THREADS) qs[d] = a.q[(int64_t)b * a.q_stride + h * HD + d];
  __syncthreads();
  const int total = a.prefix_len + len;
  auto locate = [&](int j, const Kv8View*& c) {
    const bool own = j >= a.prefix_len;
    c = own ? &a.c : &a.prefix;
    return own ? a.c.at(slot, g, j - a.prefix_len) : a.prefix.at(a.prefix_seq, g, j);
  };
  auto score = [&](int j) {
    const Kv8View* c;
    const int64_t at = locate(j, c);
    float s = 0.f;
    const char4* p = (const char4*)(c->k + at * HD);
    for (int d = 0; d < HD; d += 4) {
      const char4 w = p[d / 4];
      s += qs[d] * w.x + qs[d + 1] * w.y + qs[d + 2] * w.z + qs[d + 3] * w.w;
    }
    return s * (c->ks[at] * scale);
  };
  float m = -INFINITY;
  for (int j = threadIdx.x; j < total; j += THREADS) m = fmaxf(m, score(j));
  m = warp_max(m);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = m;
  __syncthreads();
  for (int w = 0; w < THREADS / 32; ++w) m = fmaxf(m, red[w]);
  float acc = 0.f, sum = 0.f;
  for (int j0 = 0; j0 < total; j0 += THREADS) {
    const int n = min(THREADS, total - j0);
    __syncthreads();
    if ((int)threadIdx.x < n) es[threadIdx.x] = kv8_weight(score(j0 + threadIdx.x) - m);
    __syncthreads();
    if (threadIdx.x < HD) {  // a tile's own sums first: short chains of roundings
      float ta = 0.f, ts = 0.f;
      for (int j = 0; j < n; ++j) {
        const Kv8View* c;
        const int64_t at = locate(j0 + j, c);
        ta += es[j] * ((float)c->v[at * HD + threadIdx.x] * c->vs[at]);
        ts += es[j];
      }
      acc += ta;
      sum += ts;
    }
  }
  if (threadIdx.x < HD)
    a.out[((int64_t)b * a.n_heads + h) * HD + threadIdx.x] = total > 0 ? __fdiv_rn(acc, sum) : 0.f;
}

// ---------------------------------------------------------------- decode: one cluster per (sequence, kv head)
//
// The keys are split over the cluster's CTAs, 16 keys x 8 query heads an MMA tile:
//   1. scores: K codes go from global memory into A fragments as they lie (a lane takes 16
//      neighbouring bytes of a row; q's digits, built once, are in the matching order) and the
//      scores stay in shared memory, GP floats a key;
//   2. the exact maximum of each head over the cluster (distributed shared memory);
//   3. weights e and P = e * v_scale in 23-bit fixed point against the slice's largest v_scale;
//      the three digits replace the scores in place, in B-fragment order;
//   4. out += P V: V codes become A fragments (row = dim, k = key) by 4 x 4 byte transposes;
//   5. each CTA joins its warps' sums, each rank its share of the outputs over the cluster.
// Bound by HBM at length (one pass over the codes), by the chain of phases when short.
constexpr int DT = 256;
constexpr int DW = DT / 32;

template <int HD, int GP>
struct Tile {
  static constexpr int NT = GP > 8 ? 2 : 1;     // column tiles of 8 heads
  static constexpr int CP = GP > 8 ? 8 : GP;    // heads a tile keeps
  static constexpr int KI = HD / 32;            // MMA steps of a score
  static constexpr int LD = HD / 64;            // 16-byte loads of a row a lane
  static constexpr int DS = (HD / 64) * NT;     // warps that split the dims of one key block
  static constexpr int TW = DW / DS;            // warps that split the keys
  static constexpr int DP = HD / DS;            // dims a warp
  static constexpr int MT = DP / 16;            // 16-row tiles of dims
  static constexpr int VB = DP / 8;             // bytes of a V row a lane
  // shared memory, in floats: scores | per-CTA results for the cluster
  static constexpr int PART = TW * GP * HD;     // the warps' sums take the scores' place
  static constexpr int TAIL = GP * HD + 2 * GP;
  static __host__ __device__ size_t smem_floats(int cap) {
    const int s = cap * GP;
    return (size_t)(s > PART ? s : PART) + TAIL;
  }
};

// q of one kv head's group as digits in B-fragment order; `unit` gets 2^e / sqrt(HD) of this lane's
// column head (lane / 4), the factor of its digit sums (NaN where q is not finite).
template <int HD, int GP>
__device__ __forceinline__ void load_q(const float* q, int G, int lane, uint32_t (&qd)[Tile<HD, GP>::NT][HD / 32][3][2],
                                       float (&unit)[Tile<HD, GP>::NT]) {
  using T = Tile<HD, GP>;
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) {
    const int h = nt * 8 + g;
    float x[HD / 4];
    float peak = 0.f;
#pragma unroll
    for (int l = 0; l < T::LD; ++l)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float v = h < G ? q[h * HD + l * 64 + 16 * t + i] : 0.f;
        x[l * 16 + i] = v;
        peak = max_nan(peak, fabsf(v));
      }
    peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
    peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
    const bool ok = peak < INFINITY;
    const int e = ok ? block_exp(peak) : 0;
    const float mult = pow2i(22 - e);
    unit[nt] = ok ? pow2i(e - 22) * (HD == 64 ? 0.125f : 0.0883883476f) : NAN;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const float* xs = x + 8 * i + 4 * half;
        bytes3((uint32_t)__float2int_rn(xs[0] * mult), (uint32_t)__float2int_rn(xs[1] * mult),
               (uint32_t)__float2int_rn(xs[2] * mult), (uint32_t)__float2int_rn(xs[3] * mult), qd[nt][i][0][half],
               qd[nt][i][1][half], qd[nt][i][2][half]);
      }
  }
}

template <int HD, int GP>
__global__ void __launch_bounds__(DT, (HD == 128 && GP == 16) ? 1 : 2) decode_kv8_kernel(Kv8Attn a, int cap) {
  using T = Tile<HD, GP>;
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), CL = (int)cluster.num_blocks();
  const int gk = blockIdx.y, b = blockIdx.z;
  const int G = a.n_heads / a.c.n_kv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  extern __shared__ __align__(16) float sm_[];
  float* z = sm_;                                             // [NT][cap][CP]
  float* pacc = sm_ + (T::smem_floats(cap) - T::TAIL);        // [GP][HD] this CTA's sums
  float* stat = pacc + GP * HD;                               // [GP] maximum, [GP] sum of weights
  __shared__ float wred[DW][GP], vred[DW], gmax[GP];
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int slot = a.seq_ids ? a.seq_ids[b] : b;
  if (slot < 0) return;
  const int len = a.lens[b];
  float* out = a.out + ((int64_t)b * a.n_heads + gk * G) * HD;
  if (slot >= a.c.slots || len < 0 || len > a.max_len) {
    if (tid == 0) atomicExch(a.status, SM_ERR_SHAPE);
    return;
  }
  if (len == 0) {
    if (rank == 0)
      for (int i = tid; i < G * HD; i += DT) out[i] = 0.f;
    return;
  }
  // this CTA's keys: whole blocks of 32
  const int per = ((len + CL - 1) / CL + 31) & ~31;
  const int j0 = min(len, rank * per), n = min(len - j0, per);
  const int64_t row0 = a.c.at(slot, gk, j0);
  const int8_t* kp = a.c.k + row0 * HD;
  const int8_t* vp = a.c.v + row0 * HD;
  const float* ksp = a.c.ks + row0;
  const float* vsp = a.c.vs + row0;

  // ---- 1. scores
  const int tiles = (n + 15) >> 4;
  uint4 ka[T::LD], kb[T::LD];
  float sa = 0.f, sb = 0.f;
  auto load_k = [&](int tile) {
    const int ra = min(tile * 16 + g, n - 1), rb = min(tile * 16 + 8 + g, n - 1);
#pragma unroll
    for (int l = 0; l < T::LD; ++l) {
      ka[l] = ld_codes16(kp + (int64_t)ra * HD + l * 64 + 16 * t);
      kb[l] = ld_codes16(kp + (int64_t)rb * HD + l * 64 + 16 * t);
    }
    sa = __ldg(ksp + ra);
    sb = __ldg(ksp + rb);
  };
  if (warp < tiles) load_k(warp);
  float vmax = 0.f;
  for (int j = tid; j < n; j += DT) vmax = max_nan(vmax, __ldg(vsp + j));
  uint32_t qd[T::NT][T::KI][3][2];
  float unit[T::NT];
  load_q<HD, GP>(a.q + (int64_t)b * a.q_stride + (int64_t)gk * G * HD, G, lane, qd, unit);
  float u[T::NT][2], mx[T::NT][2];  // factors and running maxima of this lane's score columns 2t, 2t + 1
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      u[nt][c] = __shfl_sync(0xffffffffu, unit[nt], (2 * t + c) * 4);
      mx[nt][c] = -INFINITY;
    }
  for (int tile = warp; tile < tiles; tile += DW) {
    uint4 ca[T::LD], cb[T::LD];
#pragma unroll
    for (int l = 0; l < T::LD; ++l) ca[l] = ka[l], cb[l] = kb[l];
    const float fa = sa, fb = sb;
    if (tile + DW < tiles) load_k(tile + DW);
    const int r = tile * 16 + g;
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) {
      int d[3][4] = {};
#pragma unroll
      for (int l = 0; l < T::LD; ++l) {
        const uint32_t* wa = (const uint32_t*)&ca[l];
        const uint32_t* wb = (const uint32_t*)&cb[l];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const auto& q3 = qd[nt][2 * l + i];
          mma_s8u8(d[0], wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], q3[0][0], q3[0][1]);
          mma_s8u8(d[1], wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], q3[1][0], q3[1][1]);
          mma_s8s8(d[2], wa[2 * i], wb[2 * i], wa[2 * i + 1], wb[2 * i + 1], q3[2][0], q3[2][1]);
        }
      }
      float s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] = join3_small(d[2][i], d[1][i], d[0][i]) * (u[nt][i & 1] * (i < 2 ? fa : fb));
      if (r < n) mx[nt][0] = fmaxf(mx[nt][0], s[0]), mx[nt][1] = fmaxf(mx[nt][1], s[1]);
      if (r + 8 < n) mx[nt][0] = fmaxf(mx[nt][0], s[2]), mx[nt][1] = fmaxf(mx[nt][1], s[3]);
      if (2 * t < T::CP) {
        float* to = z + ((int64_t)nt * cap + r) * T::CP + 2 * t;
        *(float2*)to = make_float2(s[0], s[1]);
        *(float2*)(to + 8 * T::CP) = make_float2(s[2], s[3]);
      }
    }
  }
  // the warp's first V block travels while the maxima are exchanged
  const int tw = warp / T::DS, d0 = (warp % T::DS) * T::DP;
  const int blocks = (n + 31) >> 5;
  uint32_t vw[8][T::VB / 4];
  auto load_v = [&](int blk) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int8_t* p = vp + (int64_t)min(blk * 32 + t + 4 * i, n - 1) * HD + d0 + g * T::VB;
      if constexpr (T::VB == 8) {
        const uint2 v = ld_codes8(p);
        vw[i][0] = v.x, vw[i][1] = v.y;
      } else {
        vw[i][0] = ld_codes4(p);
      }
    }
  };
  if (tw < blocks) load_v(tw);

  // ---- 2. maxima: warps, CTA, cluster
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float m = mx[nt][c];
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
      m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
      if (g == 0 && 2 * t < T::CP) wred[warp][nt * 8 + 2 * t + c] = m;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) vmax = max_nan(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
  if (lane == 0) vred[warp] = vmax;
  __syncthreads();
  if (tid < GP) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < DW; ++w) m = fmaxf(m, wred[w][tid]);
    stat[tid] = m;
  }
#pragma unroll
  for (int w = 0; w < DW; ++w) vmax = max_nan(vmax, vred[w]);
  cluster.sync();
  if (tid < GP) {
    float m = -INFINITY;
    for (int r = 0; r < CL; ++r) m = fmaxf(m, cluster.map_shared_rank(stat, r)[tid]);
    gmax[tid] = m;
  }
  __syncthreads();

  // ---- 3. weights; P in fixed point: e = 1 at the largest scale is 2^23 - 8 (scales under 1e-30 keep the
  // resolution of 1e-30, so that neither factor overflows)
  vmax = max_nan(vmax, 1e-30f);
  const float mult = 8388600.f / vmax;
  float esum[T::NT];
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) esum[nt] = 0.f;
  const int col = g < T::CP ? g : 0;
  for (int blk = warp; blk < blocks; blk += DW) {
    float vs[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) vs[i] = __ldg(vsp + min(blk * 32 + t + 4 * i, n - 1)) * mult;
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) {
      float* zb = z + ((int64_t)nt * cap + blk * 32) * T::CP;
      const float m = gmax[nt * 8 + col];
      uint32_t p[8];
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = t + 4 * i;
        float e = kv8_weight(zb[j * T::CP + col] - m);
        if (blk * 32 + j >= n) e = 0.f;
        part += e;
        // e * vs lies in [0, 2^23): added to 2^23 it is the mantissa, rounded
        p[i] = __float_as_uint(fmaf(e, vs[i], 8388608.f));
      }
      esum[nt] += part;
      uint32_t dg[3][2];
#pragma unroll
      for (int half = 0; half < 2; ++half)
        bytes3(p[4 * half], p[4 * half + 1], p[4 * half + 2], p[4 * half + 3], dg[0][half], dg[1][half], dg[2][half]);
      __syncwarp();
      if (g < T::CP) {
        uint32_t* to = (uint32_t*)zb + lane;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          to[(2 * i) * 4 * T::CP] = dg[i][0];
          to[(2 * i + 1) * 4 * T::CP] = dg[i][1];
        }
      }
    }
  }
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt) {
    esum[nt] += __shfl_xor_sync(0xffffffffu, esum[nt], 1);
    esum[nt] += __shfl_xor_sync(0xffffffffu, esum[nt], 2);
    if (t == 0 && g < T::CP) wred[warp][nt * 8 + g] = esum[nt];
  }
  __syncthreads();
  if (tid < GP) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < DW; ++w) s += wred[w][tid];
    stat[GP + tid] = s;
  }

  // ---- 4. sums of P V
  int acc[T::NT][T::MT][3][4] = {};
  for (int blk = tw; blk < blocks; blk += T::TW) {
    uint32_t w[8][T::VB / 4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int c = 0; c < T::VB / 4; ++c) w[i][c] = vw[i][c];
    if (blk + T::TW < blocks) load_v(blk + T::TW);
    uint32_t dg[T::NT][3][2];
#pragma unroll
    for (int nt = 0; nt < T::NT; ++nt) {
      const uint32_t* from = (const uint32_t*)(z + ((int64_t)nt * cap + blk * 32) * T::CP) + lane;
#pragma unroll
      for (int i = 0; i < 3; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) dg[nt][i][half] = g < T::CP ? from[(2 * i + half) * 4 * T::CP] : 0u;
    }
#pragma unroll
    for (int c = 0; c < T::VB / 4; ++c) {
      transpose4(w[0][c], w[1][c], w[2][c], w[3][c]);
      transpose4(w[4][c], w[5][c], w[6][c], w[7][c]);
    }
#pragma unroll
    for (int mt = 0; mt < T::MT; ++mt) {
      // lane's dims 2 mt, 2 mt + 1 are rows g and g + 8 of the tile
      const int c = mt >> 1, o = (mt & 1) * 2;
#pragma unroll
      for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 3; ++i)
          mma_s8u8(acc[nt][mt][i], w[o][c], w[o + 1][c], w[4 + o][c], w[4 + o + 1][c], dg[nt][i][0], dg[nt][i][1]);
    }
  }
  __syncthreads();  // the digits are read
  float* part = sm_;  // [TW][GP][HD]
  const float back = vmax * (1.f / 8388600.f);
#pragma unroll
  for (int nt = 0; nt < T::NT; ++nt)
#pragma unroll
    for (int mt = 0; mt < T::MT; ++mt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int h = nt * 8 + 2 * t + (i & 1), d = d0 + g * T::VB + 2 * mt + (i >> 1);
        if (h < G)
          part[(tw * GP + h) * HD + d] =
              join3(acc[nt][mt][2][i], acc[nt][mt][1][i], acc[nt][mt][0][i]) * back;
      }
  __syncthreads();
  for (int i = tid; i < G * HD; i += DT) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < T::TW; ++w) s += part[w * GP * HD + i];
    pacc[i] = s;
  }
  cluster.sync();
  // ---- 5. each rank its share of the outputs
  for (int i = rank * DT + tid; i < G * HD; i += CL * DT) {
    float s = 0.f, total = 0.f;
    for (int r = 0; r < CL; ++r) {
      s += cluster.map_shared_rank(pacc, r)[i];
      total += cluster.map_shared_rank(stat, r)[GP + i / HD];
    }
    out[i] = __fdiv_rn(s, total);
  }
  cluster.sync();  // no CTA's shared memory goes before the others have read it
}

constexpr size_t SMEM_MAX = 220 * 1024;

cudaLaunchConfig_t launch_config(dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster,
                                 cudaLaunchAttribute (&attr)[2]) {
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cfg;
}

// SM_ERR_UNSUPPORTED where the scores do not fit the cluster's shared memory.
template <int HD, int GP>
int launch_decode_cluster(const Kv8Attn& a, int B, int device, int sms, cudaStream_t st) {
  using T = Tile<HD, GP>;
  auto kern = decode_kv8_kernel<HD, GP>;
  cudaLaunchAttribute attr[2];
  // largest cluster that the device schedules (16 is not a portable size), found once
  static int largest[64] = {};
  if (device >= 64) return fail(SM_ERR_UNSUPPORTED, "attention_kv8: device id too large");
  if (!largest[device]) {
    SM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_MAX));
    SM_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    cudaLaunchConfig_t probe = launch_config(dim3(16), DT, SMEM_MAX, st, 16, attr);
    int fit = 0;
    const bool ok = cudaOccupancyMaxActiveClusters(&fit, (const void*)kern, &probe) == cudaSuccess && fit > 0;
    if (!ok) cudaGetLastError();
    largest[device] = ok ? 16 : 8;
  }
  int cl = largest[device];
  while (cl > 1 && (int64_t)cl * a.c.n_kv * B > 2 * sms) cl >>= 1;
  auto cap_of = [&](int c) { return ((a.max_len + c - 1) / c + 31) & ~31; };
  while (cl < largest[device] && T::smem_floats(cap_of(cl)) * 4 > SMEM_MAX) cl <<= 1;
  const size_t smem = T::smem_floats(cap_of(cl)) * 4;
  if (smem > SMEM_MAX) return SM_ERR_UNSUPPORTED;
  const cudaLaunchConfig_t cfg = launch_config(dim3(cl, a.c.n_kv, B), DT, smem, st, cl, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, a, cap_of(cl)));
  return SM_OK;
}

int launch_decode(const Kv8Attn& a, int hd, int B, int device, int sms, cudaStream_t st) {
  const int G = a.n_heads / a.c.n_kv;
  if (hd == 64)
    return G <= 4   ? launch_decode_cluster<64, 4>(a, B, device, sms, st)
           : G <= 8 ? launch_decode_cluster<64, 8>(a, B, device, sms, st)
                    : launch_decode_cluster<64, 16>(a, B, device, sms, st);
  return G <= 4   ? launch_decode_cluster<128, 4>(a, B, device, sms, st)
         : G <= 8 ? launch_decode_cluster<128, 8>(a, B, device, sms, st)
                  : launch_decode_cluster<128, 16>(a, B, device, sms, st);
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
  if (!a.prefix.k) {
    int sms = 0;
    SM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    const int rc = launch_decode(a, head_dim, B, device, sms, st);
    if (rc == SM_OK) *launches += 1;
    if (rc != SM_ERR_UNSUPPORTED) return rc;
  }
  const dim3 grid(a.n_heads, B);
  if (head_dim == 64)
    attn_kv8_kernel<64><<<grid, THREADS, 0, st>>>(a);
  else
    attn_kv8_kernel<128><<<grid, THREADS, 0, st>>>(a);
  SM_CUDA_TRY(cudaGetLastError());
  *launches += 1;
  return SM_OK;
}

int check_attn(sm_ctx* ctx, const sm_kv8* c, const float* q, int64_t q_stride, const int* seq_ids, const int* lens,
               int max_len, int B, int n_heads, const float* out, const char* what) {
  const std::string w(what);
  SM_TRY(kv8_check(c, what));
  if (B < 0 || n_heads <= 0 || n_heads % c->n_kv) return fail(SM_ERR_SHAPE, w + ": bad shape");
  if (n_heads / c->n_kv > 16) return fail(SM_ERR_UNSUPPORTED, w + ": more than 16 q heads per kv head");
  if (max_len < 0 || max_len > c->max_tokens) return fail(SM_ERR_SHAPE, w + ": max_len outside 0 .. max_tokens");
  if (q_stride < (int64_t)n_heads * c->head_dim) return fail(SM_ERR_SHAPE, w + ": q_stride is less than a row");
  if (!seq_ids && B > c->max_seqs) return fail(SM_ERR_SHAPE, w + ": more rows than slots");
  if (!ctx || (B && (!q || !lens || !out))) return fail(SM_ERR_INVALID_ARG, w + ": null argument");
  if (((uintptr_t)q | (uintptr_t)out) % 4) return fail(SM_ERR_INVALID_ARG, w + ": misaligned pointer");
  return SM_OK;
}

}  // namespace
}  // namespace sm

using namespace sm;

extern "C" {

SM_API int sm_attention_decode_kv8(sm_ctx* ctx, const sm_kv8* cache, const float* q, int64_t q_stride,
                                   const int* seq_ids, const int* lens, int max_len, int B, int n_heads,
                                   float* out) {
  const char* what = "attention_decode_kv8";
  SM_TRY(check_attn(ctx, cache, q, q_stride, seq_ids, lens, max_len, B, n_heads, out, what));
  if (B == 0) return SM_OK;
  Kv8Attn a{kv8_view(cache), {}, 0, 0, q, q_stride, seq_ids, lens, max_len, n_heads, out, nullptr};
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
            out, nullptr};
  return attend(ctx, a, cache->head_dim, B, what);
}

}  // extern "C"
