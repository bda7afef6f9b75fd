// Decode attention of a batch behind a shared prefix, over the 8-bit KV cache, on tcgen05.
//
// The batch's query rows of one kv head (B * group of them) are the rows of a matrix product with the
// prefix's keys, which is what makes the prefix worth reading once.  Formulas as in attn_kv8.cu; the exact
// maximum over the prefix and the own keys comes first, so the scores are formed twice:
//   prep    K codes -> fp16 tiles, V codes -> transposed fp16 tiles (codes are exact in fp16), query rows,
//           scaled by a power of two into [-1, 1], -> fp16 pairs hi + lo (22 bits);
//   max     S = (hi + lo) K^T per tile of 128 rows and block of 128 keys; row maxima of S * k_scale;
//   own     (attn_kv8.cu) scores and maxima of the sequences' own keys;
//   P V     S again, e against the maximum of both parts, P = e * v_scale relative to the chunk's largest
//           scale as fp16 pairs hi + lo, O += (hi + lo) V;
//   own     P V of the own keys;
//   join    the chunks' sums and weights, in order.
// All products run as kind::f16 MMAs into fp32 TMEM accumulators; P goes back to TMEM over the scores it came
// from and is the A operand from there.  Two score buffers: while the softmax warps work on one block, the
// tensor cores form the next block's scores and the last block's P V.  Bound by the softmax arithmetic
// (about 16 instructions a score) in the P V pass, by shared-memory reads of the MMAs in the max pass.
#include <cuda_fp16.h>

#include <algorithm>

#include "kv8.cuh"
#include "kv8_mma.cuh"
#include "mbar.cuh"

namespace sm {
namespace {

constexpr int QB = 128;         // query rows of a tile
constexpr int KB = 128;         // keys of a block
constexpr int SOFT_WARPS = 8;   // TMEM lane quarter = warp % 4, key half = warp / 4
constexpr int LOAD_WARP = SOFT_WARPS, MMA_WARP = SOFT_WARPS + 1;
constexpr int THREADS = (SOFT_WARPS + 2) * 32;
constexpr int MAX_CHUNK = 28;   // blocks of a chunk, for which the scales have room in shared memory
constexpr int TMEM_COLS = 512;
constexpr uint32_t TM_S = 0, TM_O = 256;  // two score buffers of 128 columns, then O

struct SharedArgs {
  Kv8Attn a;
  int rows, tiles;          // query rows of a kv head, tiles of 128
  int n_blocks;             // blocks of 128 keys
  int chunk, n_chunks;      // blocks of a chunk
  uint8_t *kt, *vt;         // [n_kv][n_blocks] fp16 tiles [128 keys][HD] / [HD][128 keys]
  uint8_t* qt;              // [n_kv][tiles][hi | lo] fp16 tiles [128 rows][HD]
  float* unit;              // [n_kv][tiles * 128] factor of a row's scores
  float* row_max;           // [n_kv][n_chunks][tiles * 128]
  float* acc;               // [n_kv][n_chunks][tiles * 128][HD]
  float* sum;               // [n_kv][n_chunks][tiles * 128]
  Kv8Split own;             // the own keys (own.n_chunks == 0: none)
};

// ---------------------------------------------------------------- tcgen05 pieces
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// K-major operand, 128-byte swizzle, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t sw128_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// byte offset of 16-byte chunk c of row r in a column of 128-byte swizzle atoms
__host__ __device__ __forceinline__ uint32_t sw_off(int r, int c) {
  return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}
// kind::f16, fp32 accumulator, fp16 A and B, both K-major, M = 128, N = n
__host__ __device__ constexpr uint32_t idesc(int n) {
  return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
// A from TMEM: lane = row, a 32-bit column holds two neighbouring k
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// the softmax warps alone
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SOFT_WARPS * 32) : "memory"); }

// Four int8 codes as two fp16 pairs: 0x6400 + (code + 128) is 1024 + code + 128
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  w ^= 0x80808080u;
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 x = __hsub2(*(const __half2*)&a, bias), y = __hsub2(*(const __half2*)&b, bias);
  lo = *(const uint32_t*)&x;
  hi = *(const uint32_t*)&y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}

// ---------------------------------------------------------------- prep
// Blocks of the grid: K tiles, V tiles, query tiles.  Keys past the prefix and rows past the batch are zeros.
template <int HD>
__global__ void __launch_bounds__(256) shared_prep_kernel(SharedArgs s) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Kv8Attn& a = s.a;
  const int tid = threadIdx.x;
  const int n_kt = a.c.n_kv * s.n_blocks;
  int id = blockIdx.x;
  if (id < 2 * n_kt) {
    const bool is_v = id >= n_kt;
    if (is_v) id -= n_kt;
    const int g = id / s.n_blocks, blk = id - g * s.n_blocks;
    const int n = min(KB, a.prefix_len - blk * KB);
    const int8_t* src = (is_v ? a.prefix.v : a.prefix.k) + a.prefix.at(a.prefix_seq, g, blk * KB) * HD;
    uint8_t* dst = (is_v ? s.vt : s.kt) + (int64_t)id * (KB * HD * 2);
    if (!is_v) {
      for (int i = tid; i < KB * HD / 8; i += 256) {
        const int r = i / (HD / 8), c = i % (HD / 8);
        const uint2 w = r < n ? *(const uint2*)(src + r * HD + c * 8) : make_uint2(0, 0);
        uint4 o;
        codes_to_half(w.x, o.x, o.y);
        codes_to_half(w.y, o.z, o.w);
        *(uint4*)(dst + (c >> 3) * (KB * 128) + sw_off(r, c & 7)) = o;
      }
      return;
    }
    __shared__ uint8_t tile[KB][HD + 4];
    for (int i = tid; i < KB * HD / 4; i += 256) {
      const int r = i / (HD / 4), c = i % (HD / 4);
      *(uint32_t*)&tile[r][4 * c] = r < n ? *(const uint32_t*)(src + r * HD + 4 * c) : 0u;
    }
    __syncthreads();
    for (int i = tid; i < HD * KB / 8; i += 256) {
      const int d = i / (KB / 8), c = i % (KB / 8);  // dim, chunk of 8 keys
      uint32_t w[2];
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[h] = (uint32_t)tile[8 * c + 4 * h][d] | (uint32_t)tile[8 * c + 4 * h + 1][d] << 8 |
               (uint32_t)tile[8 * c + 4 * h + 2][d] << 16 | (uint32_t)tile[8 * c + 4 * h + 3][d] << 24;
      uint4 o;
      codes_to_half(w[0], o.x, o.y);
      codes_to_half(w[1], o.z, o.w);
      *(uint4*)(dst + (c >> 3) * (HD * 128) + sw_off(d, c & 7)) = o;
    }
    return;
  }
  id -= 2 * n_kt;
  const int g = id / s.tiles, tile = id - g * s.tiles;
  const int G = a.n_heads / a.c.n_kv, lane = tid & 31;
  uint8_t* dst = s.qt + (int64_t)id * (2 * QB * HD * 2);
  constexpr int E = HD / 32;  // dims a lane
  for (int r = tid >> 5; r < QB; r += 8) {
    const int row = tile * QB + r;
    const int b = row / G, h = row - b * G;
    const bool live = row < s.rows && (!a.seq_ids || a.seq_ids[b] >= 0);
    const float* q = a.q + (int64_t)b * a.q_stride + (int64_t)(g * G + h) * HD + E * lane;
    float x[E];
    float peak = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = live ? q[i] : 0.f, peak = max_nan(peak, fabsf(x[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    const bool ok = peak < INFINITY;
    const int e = ok ? block_exp(peak) : 0;
    const float mult = pow2i(-e);
    if (lane == 0)
      s.unit[(int64_t)id * QB + r] = ok ? pow2i(e) * (HD == 64 ? 0.125f : 0.0883883476f) : NAN;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float y0 = ok ? x[i] * mult : 0.f, y1 = ok ? x[i + 1] * mult : 0.f;
      const uint32_t hi = pack_half(y0, y1);
      const float2 f = __half22float2(*(const __half2*)&hi);
      const int d = E * lane + i;
      uint8_t* p = dst + (d >> 6) * (QB * 128) + sw_off(r, (d & 63) >> 3) + (d & 7) * 2;
      *(uint32_t*)p = hi;
      *(uint32_t*)(p + QB * HD * 2) = pack_half(y0 - f.x, y1 - f.y);
    }
  }
}

// ---------------------------------------------------------------- the two passes
template <int HD>
struct TcSmem {
  static constexpr int TILE = 128 * HD * 2;  // bytes of any tile
  static constexpr int Q = 0, K = Q + 2 * TILE, V = K + 2 * TILE, SCALES = V + 2 * TILE;
  static constexpr int BARS = SCALES + 2 * MAX_CHUNK * KB * 4;
  static constexpr size_t BYTES = (size_t)BARS + 256 + 1024;  // and alignment slack
};

// MAX: grid (n_chunks, tiles, n_kv): row maxima of S * k_scale.  Else: the chunk's O and weight sums.
template <int HD, bool MAX>
__global__ void __launch_bounds__(THREADS, 1) shared_pass_kernel(const __grid_constant__ SharedArgs s) {
  using M = TcSmem<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bar = (uint64_t*)(smem + M::BARS);
  uint64_t* q_full = bar;
  uint64_t* k_full = bar + 1;    // [2]
  uint64_t* v_full = bar + 3;    // [2]
  uint64_t* s_full = bar + 5;    // [2] scores formed; the K slot is free
  uint64_t* s_done = bar + 7;    // [2] MAX: scores read; else: P written
  uint64_t* pv_done = bar + 9;   // [2] P V formed; the V slot and the score buffer are free
  uint32_t* tmem_slot = (uint32_t*)(bar + 11);
  float* ks = (float*)(smem + M::SCALES);
  float* vs = ks + MAX_CHUNK * KB;
  const Kv8Attn& a = s.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ch = blockIdx.x, tile = blockIdx.y, g = blockIdx.z;
  const int blk0 = ch * s.chunk, nb = min(s.chunk, s.n_blocks - blk0);
  const int64_t rows = (int64_t)s.tiles * QB;

  if (tid == 0) {
    mbar_init(q_full, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&s_done[i], SOFT_WARPS * 32);
      mbar_init(&pv_done[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == LOAD_WARP) {
    if (lane == 0) {
      const uint8_t* q = s.qt + ((int64_t)g * s.tiles + tile) * (2 * M::TILE);
      mbar_expect_tx(q_full, 2 * M::TILE);
      bulk_g2s(smem + M::Q, q, M::TILE, q_full);
      bulk_g2s(smem + M::Q + M::TILE, q + M::TILE, M::TILE, q_full);
      const int64_t first = (int64_t)g * s.n_blocks + blk0;
      for (int j = 0; j < nb; ++j) {
        const int i = j & 1, use = (j >> 1) - 1;
        if (use >= 0 && !mbar_wait_bounded(&s_full[i], use & 1, a.status)) break;
        mbar_expect_tx(&k_full[i], M::TILE);
        bulk_g2s(smem + M::K + i * M::TILE, s.kt + (first + j) * M::TILE, M::TILE, &k_full[i]);
        if (!MAX) {
          if (use >= 0 && !mbar_wait_bounded(&pv_done[i], use & 1, a.status)) break;
          mbar_expect_tx(&v_full[i], M::TILE);
          bulk_g2s(smem + M::V + i * M::TILE, s.vt + (first + j) * M::TILE, M::TILE, &v_full[i]);
        }
      }
    }
  } else if (warp == MMA_WARP) {
    if (lane == 0) {
      const uint32_t qa = smem_u32(smem + M::Q), ka = smem_u32(smem + M::K), va = smem_u32(smem + M::V);
      bool ok = mbar_wait_bounded(q_full, 0, a.status);
      auto scores = [&](int j) {
        const int i = j & 1, use = j >> 1;
        ok = ok && mbar_wait_bounded(&k_full[i], use & 1, a.status);
        if (use > 0) ok = ok && mbar_wait_bounded(MAX ? &s_done[i] : &pv_done[i], (use - 1) & 1, a.status);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int ks16 = 0; ks16 < HD / 16; ++ks16) {
          const uint32_t at = (uint32_t)((ks16 >> 2) * (128 * 128) + (ks16 & 3) * 32);
          const uint64_t k = sw128_desc(ka + i * M::TILE + at);
          mma_ss(tmem + TM_S + i * KB, sw128_desc(qa + at), k, idesc(KB), ks16 != 0);
          mma_ss(tmem + TM_S + i * KB, sw128_desc(qa + M::TILE + at), k, idesc(KB), 1);
        }
        mma_commit(&s_full[i]);
      };
      scores(0);
      if (nb > 1) scores(1);
      for (int j = 0; j < nb && ok; ++j) {
        const int i = j & 1, use = j >> 1;
        if (!MAX) {
          ok = mbar_wait_bounded(&v_full[i], use & 1, a.status) && mbar_wait_bounded(&s_done[i], use & 1, a.status);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks16 = 0; ks16 < KB / 16; ++ks16) {
            // keys 16 ks16 ..: P hi, then lo, in the score columns of their 32 keys
            const uint32_t p = tmem + TM_S + i * KB + (ks16 >> 1) * 32 + (ks16 & 1) * 8;
            const uint64_t v =
                sw128_desc(va + i * M::TILE + (uint32_t)((ks16 >> 2) * (HD * 128) + (ks16 & 3) * 32));
            mma_ts(tmem + TM_O, p, v, idesc(HD), (j | ks16) != 0);
            mma_ts(tmem + TM_O, p + 16, v, idesc(HD), 1);
          }
          mma_commit(&pv_done[i]);
        }
        if (j + 2 < nb) scores(j + 2);
      }
    }
  } else {
    const int r = (warp & 3) * 32 + lane, half = warp >> 2;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const int64_t row = (int64_t)g * rows + tile * QB + r;
    // the chunk's scales; a key past the prefix gets NaN (MAX: no maximum takes it) or 0
    const int64_t at = a.prefix.at(a.prefix_seq, g, blk0 * KB);
    const int keys = min(nb * KB, a.prefix_len - blk0 * KB);
    float vmax = 0.f;
    for (int j = tid; j < nb * KB; j += SOFT_WARPS * 32) {
      ks[j] = j < keys ? __ldg(a.prefix.ks + at + j) : MAX ? NAN : 0.f;
      if (!MAX) {
        const float v = j < keys ? __ldg(a.prefix.vs + at + j) : 0.f;
        vs[j] = v;
        vmax = max_nan(vmax, v);
      }
    }
    bool ok = true;
    if constexpr (MAX) {
      soft_sync();
      float m = -INFINITY;
      for (int j = 0; j < nb && ok; ++j) {
        const int i = j & 1;
        ok = mbar_wait_bounded(&s_full[i], (j >> 1) & 1, a.status);
        tc_fence_after();
        uint32_t x[2][32];
        tmem_ld32(trow + TM_S + i * KB + half * 64, x[0]);
        tmem_ld32(trow + TM_S + i * KB + half * 64 + 32, x[1]);
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(&s_done[i]);
        const float4* k4 = (const float4*)(ks + j * KB + half * 64);
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 k = k4[(32 * c + e) / 4];
            m = fmaxf(m, fmaxf(__uint_as_float(x[c][e]) * k.x, __uint_as_float(x[c][e + 1]) * k.y));
            m = fmaxf(m, fmaxf(__uint_as_float(x[c][e + 2]) * k.z, __uint_as_float(x[c][e + 3]) * k.w));
          }
      }
      soft_sync();  // the scales are read
      if (half) ks[r] = m;
      soft_sync();
      if (!half) s.row_max[((int64_t)g * s.n_chunks + ch) * rows + tile * QB + r] = fmaxf(m, ks[r]) * s.unit[row];
    } else {
      // the largest V scale of the chunk, by way of O's slot in shared memory
      __shared__ float red[SOFT_WARPS];
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) vmax = max_nan(vmax, __shfl_xor_sync(0xffffffffu, vmax, o));
      if (lane == 0) red[warp] = vmax;
      soft_sync();
#pragma unroll
      for (int i = 0; i < SOFT_WARPS; ++i) vmax = max_nan(vmax, red[i]);
      vmax = max_nan(vmax, 1e-30f);  // under it P keeps the resolution of 1e-30
      const float mult = 1.f / vmax;
      for (int j = tid; j < nb * KB; j += SOFT_WARPS * 32) vs[j] *= mult;
      // the row's maximum over the prefix's chunks and the own ones
      const float unit = s.unit[row];
      float m = -INFINITY;
      for (int c = 0; c < s.n_chunks; ++c)
        m = fmaxf(m, __ldg(s.row_max + ((int64_t)g * s.n_chunks + c) * rows + tile * QB + r));
      if (s.own.n_chunks && tile * QB + r < s.rows) {
        const int G = a.n_heads / a.c.n_kv, b = (tile * QB + r) / G, h = (tile * QB + r) % G;
        const int slot = a.seq_ids ? a.seq_ids[b] : b, len = a.lens[b];
        if (slot >= 0 && slot < a.c.slots && len >= 0 && len <= a.max_len) {
          const int used = (len + s.own.chunk - 1) / s.own.chunk;
          const float* st = s.own.stat + ((int64_t)b * a.c.n_kv + g) * s.own.n_chunks * (2 * s.own.gp + 1) + h;
          for (int c = 0; c < used; ++c) m = fmaxf(m, st[c * (2 * s.own.gp + 1)] * (unit * (1.f / 4194304.f)));
        }
      }
      soft_sync();
      float sum = 0.f;
      for (int j = 0; j < nb && ok; ++j) {
        const int i = j & 1;
        ok = mbar_wait_bounded(&s_full[i], (j >> 1) & 1, a.status);
        tc_fence_after();
        const uint32_t cols = trow + TM_S + i * KB + half * 64;
        const int left = keys - j * KB - half * 64;  // keys of this thread's 64 that exist
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t x[32];
          tmem_ld32(cols + 32 * c, x);
          tmem_wait_ld();
          const float4* k4 = (const float4*)(ks + j * KB + half * 64 + 32 * c);
          const float4* v4 = (const float4*)(vs + j * KB + half * 64 + 32 * c);
          uint32_t hi[16], lo[16];
          float part = 0.f;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            const float4 k = k4[e / 4], v = v4[e / 4];
            float w[4];
            w[0] = kv8_weight(fmaf(__uint_as_float(x[e]) * k.x, unit, -m));
            w[1] = kv8_weight(fmaf(__uint_as_float(x[e + 1]) * k.y, unit, -m));
            w[2] = kv8_weight(fmaf(__uint_as_float(x[e + 2]) * k.z, unit, -m));
            w[3] = kv8_weight(fmaf(__uint_as_float(x[e + 3]) * k.w, unit, -m));
            if (left < 64) {
#pragma unroll
              for (int o = 0; o < 4; ++o)
                if (32 * c + e + o >= left) w[o] = 0.f;
            }
            part += (w[0] + w[1]) + (w[2] + w[3]);
            const float p0 = w[0] * v.x, p1 = w[1] * v.y, p2 = w[2] * v.z, p3 = w[3] * v.w;
            hi[e / 2] = pack_half(p0, p1);
            hi[e / 2 + 1] = pack_half(p2, p3);
            const float2 f0 = __half22float2(*(const __half2*)&hi[e / 2]);
            const float2 f1 = __half22float2(*(const __half2*)&hi[e / 2 + 1]);
            lo[e / 2] = pack_half(p0 - f0.x, p1 - f0.y);
            lo[e / 2 + 1] = pack_half(p2 - f1.x, p3 - f1.y);
          }
          sum += part;
          tmem_st16(cols + 32 * c, hi);
          tmem_st16(cols + 32 * c + 16, lo);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&s_done[i]);
      }
      // O: the last P V is done, and with it all of them
      ok = ok && mbar_wait_bounded(&pv_done[(nb - 1) & 1], ((nb - 1) >> 1) & 1, a.status);
      tc_fence_after();
      soft_sync();  // the scales are read
      ks[half * QB + r] = sum;
      soft_sync();
      const int64_t out = ((int64_t)g * s.n_chunks + ch) * rows + tile * QB + r;
      if (!half) s.sum[out] = ks[r] + ks[QB + r];
#pragma unroll
      for (int c = 0; c < HD / 64; ++c) {
        uint32_t x[32];
        tmem_ld32(trow + TM_O + half * (HD / 2) + 32 * c, x);
        tmem_wait_ld();
        float* o = s.acc + out * HD + half * (HD / 2) + 32 * c;
        if (ok) {
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            *(float4*)(o + e) =
                make_float4(__uint_as_float(x[e]) * vmax, __uint_as_float(x[e + 1]) * vmax,
                            __uint_as_float(x[e + 2]) * vmax, __uint_as_float(x[e + 3]) * vmax);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

// grid (n_heads, B), HD threads
__global__ void shared_join_kernel(SharedArgs s) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Kv8Attn& a = s.a;
  const int head = blockIdx.x, b = blockIdx.y, d = threadIdx.x, HD = blockDim.x;
  int slot, len;
  if (!row_keys(a, b, slot, len)) return;
  const int G = a.n_heads / a.c.n_kv, g = head / G, h = head - g * G;
  const int64_t rows = (int64_t)s.tiles * QB;
  float x = 0.f, total = 0.f;
#pragma unroll 4
  for (int c = 0; c < s.n_chunks; ++c) {
    const int64_t row = ((int64_t)g * s.n_chunks + c) * rows + (int64_t)b * G + h;
    x += s.acc[row * HD + d];
    total += s.sum[row];
  }
  if (s.own.n_chunks) {
    const int used = (len + s.own.chunk - 1) / s.own.chunk, gp = s.own.gp;
    const int64_t row = ((int64_t)b * a.c.n_kv + g) * s.own.n_chunks;
    for (int c = 0; c < used; ++c) {
      x += s.own.pacc[((row + c) * gp + h) * HD + d];
      total += s.own.stat[(row + c) * (2 * gp + 1) + gp + 1 + h];
    }
  }
  a.out[((int64_t)b * a.n_heads + head) * HD + d] = __fdiv_rn(x, total);
}

template <int HD>
int launch_shared(SharedArgs& s, int B, cudaStream_t st, int* n_launch) {
  using M = TcSmem<HD>;
  auto max_pass = shared_pass_kernel<HD, true>;
  auto pv_pass = shared_pass_kernel<HD, false>;
  SM_CUDA_TRY(cudaFuncSetAttribute(max_pass, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)M::BYTES));
  SM_CUDA_TRY(cudaFuncSetAttribute(pv_pass, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)M::BYTES));
  cudaLaunchAttribute attr[2];
  const int n_kv = s.a.c.n_kv;
  cudaLaunchConfig_t cfg = launch_config(dim3(2 * n_kv * s.n_blocks + n_kv * s.tiles), 256, 0, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, shared_prep_kernel<HD>, s));
  const dim3 grid(s.n_chunks, s.tiles, n_kv);
  cfg = launch_config(grid, THREADS, M::BYTES, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, max_pass, s));
  *n_launch += 2;
  if (s.own.n_chunks) {
    SM_TRY(launch_kv8_split_scores(s.own, HD, B, st));
    ++*n_launch;
  }
  cfg = launch_config(grid, THREADS, M::BYTES, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, pv_pass, s));
  ++*n_launch;
  if (s.own.n_chunks) {
    SM_TRY(launch_kv8_split_pv(s.own, HD, B, st));
    ++*n_launch;
  }
  cfg = launch_config(dim3(s.a.n_heads, B), HD, 0, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, shared_join_kernel, s));
  ++*n_launch;
  return SM_OK;
}

}  // namespace

int launch_attention_shared_tc(const Kv8Attn& a, int hd, int B, int sms, cudaStream_t st, int* n_launch) {
  SharedArgs s = {};
  s.a = a;
  const int n_kv = a.c.n_kv;
  const int64_t rows = (int64_t)B * (a.n_heads / n_kv);
  if (rows > INT32_MAX - QB) return fail(SM_ERR_SHAPE, "attention_shared_kv8: batch too large");
  s.rows = (int)rows;
  s.tiles = ceil_div(rows, QB);
  s.n_blocks = ceil_div(a.prefix_len, KB);
  if (s.tiles > 65535 || n_kv > 65535 || 2ll * n_kv * s.n_blocks + (int64_t)n_kv * s.tiles > INT32_MAX)
    return fail(SM_ERR_SHAPE, "attention_shared_kv8: batch too large");
  // chunks of at most MAX_CHUNK blocks, as many as make the fewest block times over the waves of CTAs; a CTA's
  // start and end cost about 3 blocks
  const int64_t ctas = (int64_t)s.tiles * n_kv;
  int64_t best = INT64_MAX;
  for (int n = ceil_div(s.n_blocks, MAX_CHUNK); n <= std::min(s.n_blocks, ceil_div(s.n_blocks, MAX_CHUNK) + 64); ++n) {
    const int chunk = ceil_div(s.n_blocks, n);
    const int64_t cost = (ctas * ceil_div(s.n_blocks, chunk) + sms - 1) / sms * (chunk + 3);
    if (cost < best) best = cost, s.chunk = chunk;
  }
  s.n_chunks = ceil_div(s.n_blocks, s.chunk);
  s.own.a = a;
  const int64_t tile = 128ll * hd * 2, rp = ctas * QB;
  const int64_t kv_bytes = n_kv * (int64_t)s.n_blocks * tile, q_bytes = ctas * 2 * tile;
  const int64_t floats = rp + rp * s.n_chunks * (2 + hd);
  const int64_t own = a.max_len > 0 ? kv8_split_plan(s.own, hd, B, sms) : 0;
  uint8_t* buf = nullptr;
  if (cudaMallocAsync((void**)&buf, (size_t)(2 * kv_bytes + q_bytes + (floats + own) * 4), st) != cudaSuccess) {
    cudaGetLastError();
    return fail(SM_ERR_OOM, "attention_shared_kv8: device allocation failed");
  }
  s.kt = buf;
  s.vt = s.kt + kv_bytes;
  s.qt = s.vt + kv_bytes;
  s.acc = (float*)(s.qt + q_bytes);
  s.unit = s.acc + rp * s.n_chunks * hd;
  s.row_max = s.unit + rp;
  s.sum = s.row_max + rp * s.n_chunks;
  if (own) {
    kv8_split_place(s.own, hd, B, s.sum + rp * s.n_chunks);
    s.own.prefix_max = s.row_max;
    s.own.prefix_chunks = s.n_chunks;
    s.own.prefix_rows = s.tiles * QB;
  }
  const int rc = hd == 64 ? launch_shared<64>(s, B, st, n_launch) : launch_shared<128>(s, B, st, n_launch);
  cudaFreeAsync(buf, st);
  return rc;
}

}  // namespace sm
