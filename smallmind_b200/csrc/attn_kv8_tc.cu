// Decode attention of a batch behind a shared prefix, over the 8-bit KV cache, on tcgen05.
//
// The batch's query rows of one kv head (B * group of them) are the rows of a matrix product with the
// prefix's keys, which is what makes the prefix worth reading once.  Formulas as in attn_kv8.cu; the exact
// maximum over the prefix and the own keys comes first, so the scores are formed twice:
//   prep    K and V codes -> fp16 tiles (codes are exact in fp16), query rows, scaled by a power of two into
//           [-1, 1], -> fp16 pairs hi + lo (22 bits);
//   max     S = (hi + lo) K^T per tile of 128 rows and block of 128 keys; row maxima of the scores S * (k_scale *
//           the row's factor): the factors meet first, or S times a large scale would leave fp32's range;
//   own     (attn_kv8.cu) the sequences' own keys, against the maximum of both parts;
//   P V     S again, e against the maximum of both parts, P = e * v_scale relative to the prefix's largest
//           scale as fp16 pairs hi + lo, O += (hi + lo) V;
//   join    the parts' sums and weights, in order.
// All products run as kind::f16 MMAs into fp32 TMEM accumulators; A (the query rows, then P, which takes the
// place of the scores it came from) is in TMEM.  K and V tiles are laid out alike, in 128-byte-swizzled rows of
// a key, and come by one bulk copy each (K as a K-major B operand, V as an MN-major one).  While the softmax
// warps work on one block, the tensor cores form the next block's scores and the last block's P V.  The (row
// tile, block) units are dealt evenly to one CTA an SM, so that CTAs with different row tiles walk the same blocks
// together (they then come from L2: with 8 tiles of rows, each by itself, 747 MB came from HBM instead of 144); a
// CTA's units of one tile make a segment with sums of its own.  The accumulation of O inside the tensor cores
// truncates: over 111 blocks it was 2e-5 off, so every FLUSH blocks O moves on to fp32 sums in memory.
//
// q and P as fp16 pairs hold 22 bits of a row's largest |q| and of the prefix's largest V scale, where fp32 holds 24 of
// each value; a third half would be half as many MMAs again.
//
// Bound by the tensor cores: a block takes 16 + 32 MMAs (head_dim 128) in the two passes, 64 clocks each (counted:
// the cycles in which the tensor pipe is active, over the MMAs of a CTA, in both passes).  32 / 8 heads of 128, 256
// rows over 32768 keys, each kernel alone and with cold caches: max 98 us (84 % of the time on the tensor pipe), P V
// 225 us (70 %: P of a block is waited for while both score buffers are taken), both at an SM clock of 1.60 GHz; prep
// 34 us (HBM: 67 MB of codes in, 134 MB of tiles out), own keys 50 us, join 12 us; the whole call, whose launches
// overlap, 377 us.  Tried when P V took 218 us: four score buffers of 64 keys keep the pipe full, but an MMA of 64
// columns takes as long as one of 128 (238 us); two halves of the softmax warps that take every other block 230 us; 8
// softmax warps instead of 16 the same time.
#include <cuda_fp16.h>

#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "kv8_mma.cuh"
#include "mbar.cuh"

namespace sm {
namespace {

constexpr int QB = 128;          // query rows of a tile
constexpr int KB = 128;          // keys of a block
constexpr int SOFT_WARPS = 16;   // TMEM lane quarter = warp % 4, keys of a block: part warp / 4
constexpr int SOFT = SOFT_WARPS * 32;
constexpr int PARTS = SOFT_WARPS / 4;
constexpr int PK = KB / PARTS;   // keys of a part
constexpr int LOAD_WARP = SOFT_WARPS, MMA_WARP = SOFT_WARPS + 1;
constexpr int THREADS = SOFT + 64;
constexpr int NSC = 4;           // ring slots of block scales
constexpr int FLUSH = 16;        // blocks that O accumulates in TMEM
constexpr int TMEM_COLS = 512;
constexpr uint32_t TM_S = 0, TM_O = 256, TM_Q = 384;  // score buffers of 128 columns, O, query rows hi and lo

struct SharedArgs {
  Kv8Attn a;
  int rows, tiles;          // query rows of a kv head, tiles of 128
  int n_blocks;             // blocks of 128 keys
  // Units (tile, block) are dealt to groups of `ways` CTAs, which walk the same blocks at the same time with
  // neighbouring tiles: a line of blocks belongs to `ways` tiles.  The lines lie behind one another, n_blocks each.
  int ways, units;          // a divisor of tiles; blocks of all lines
  int per, n_ctas;          // blocks of a CTA; CTAs
  uint8_t *kt, *vt;         // [n_kv][n_blocks] fp16 tiles [128 keys][HD]
  float* scales;            // [n_kv][n_blocks][K 128 | V 128]; past the prefix NaN | 0
  uint8_t* qt;              // [n_kv][tiles][hi | lo][128 rows][HD] fp16
  float* unit;              // [n_kv][tiles * 128] factor of a row's scores
  float* row_max;           // [n_kv][tiles * 128] largest score over the prefix
  float* v_max;             // [n_kv][n_blocks][4] largest V scales of 32 keys each
  float* v_top;             // [n_kv] the head's largest, at least 2^-126
  float* acc;               // [segment][128][HD]; segment = CTA + tile of all kv heads, in lines (segment_of)
  float* sum;               // [segment][128]
  float* own_max;           // [n_kv][tiles * 128] largest own score, -inf where there is none
  float* own_acc;           // [n_kv][tiles * 128][HD] the own keys' part; nullptr: nobody has any
  float* own_sum;           // [n_kv][tiles * 128]
};

// A group's sums for a line of blocks, of one of its tiles; the groups and the lines both ascend, so no two share one
__device__ __forceinline__ int64_t segment_of(const SharedArgs& s, int group, int line, int way) {
  return ((int64_t)group + line) * s.ways + way;
}

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
// MN-major operand, 128-byte swizzle: 8 rows of k 1024 bytes apart, 64 columns of n 128 rows apart
__device__ __forceinline__ uint64_t sw128_desc_mn(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(KB * 128 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// kind::f16, fp32 accumulator, fp16 A and B, A K-major, M = 128, N = n; b_mn: B is MN-major
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
// One lane of a converged warp.  The MMA warp runs as a whole and only the instructions themselves are left to
// one lane: their operands then stay in uniform registers (issued from a one-lane branch, an MMA took 66 to 80
// clocks to issue, which bound both passes).
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// A from TMEM: lane = row, a 32-bit column holds two neighbouring k
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t acc) {
  if (elect())
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if (elect())
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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// The loads of r have arrived.  r passes through, so that nothing that uses it can be moved ahead of the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                 "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                 "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                 "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Shared memory that bulk copies write again: a plain load was seen to be moved past the arrival that frees it
__device__ __forceinline__ float4 ld_slot(uint32_t at) {
  float4 v;
  asm volatile("ld.volatile.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(at)
               : "memory");
  return v;
}
// the softmax warps alone
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(SOFT) : "memory"); }

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
// Blocks of the grid: K tiles, V tiles, parts of 16 rows of the query tiles.  Keys past the prefix and rows past
// the batch are zeros.
template <int HD>
__global__ void __launch_bounds__(256) shared_prep_kernel(SharedArgs s) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Kv8Attn& a = s.a;
  const int tid = threadIdx.x, lane = tid & 31;
  const int n_kt = a.c.n_kv * s.n_blocks;
  int id = blockIdx.x;
  if (id < 2 * n_kt) {
    const bool is_v = id >= n_kt;
    if (is_v) id -= n_kt;
    const int g = id / s.n_blocks, blk = id - g * s.n_blocks;
    const int n = min(KB, a.prefix_len - blk * KB);
    const int64_t at = a.prefix.at(a.prefix_seq, g, blk * KB);
    const int8_t* src = (is_v ? a.prefix.v : a.prefix.k) + at * HD;
    uint8_t* dst = (is_v ? s.vt : s.kt) + (int64_t)id * (KB * HD * 2);
    // 8 codes a thread and step; a warp's stores fill whole lines
    constexpr int C = HD / 8, STEPS = KB * C / 256;
    const int c = tid % C, r0 = tid / C;
    uint2 x[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int r = r0 + i * (256 / C);
      x[i] = r < n ? *(const uint2*)(src + r * HD + c * 8) : make_uint2(0, 0);
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      uint4 o;
      codes_to_half(x[i].x, o.x, o.y);
      codes_to_half(x[i].y, o.z, o.w);
      *(uint4*)(dst + (c >> 3) * (KB * 128) + sw_off(r0 + i * (256 / C), c & 7)) = o;
    }
    if (tid < KB) {
      const float sc = tid < n ? (is_v ? a.prefix.vs : a.prefix.ks)[at + tid] : is_v ? 0.f : NAN;
      s.scales[(int64_t)id * (2 * KB) + is_v * KB + tid] = sc;
      if (is_v) {
        float m = sc;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) s.v_max[id * 4 + (tid >> 5)] = m;
      }
    }
    return;
  }
  id -= 2 * n_kt;
  const int part = id % (QB / 16);
  id /= QB / 16;
  const int g = id / s.tiles, tile = id - g * s.tiles;
  const int G = a.n_heads / a.c.n_kv;
  uint8_t* dst = s.qt + (int64_t)id * (2 * QB * HD * 2);
  constexpr int E = HD / 32;  // dims a lane
  for (int r = part * 16 + (tid >> 5); r < part * 16 + 16; r += 8) {
    const int row = tile * QB + r;
    const int b = row / G, h = row - b * G;
    const bool live = row < s.rows && row_in_range(a, b);
    const float* q = a.q + (int64_t)b * a.q_stride + (int64_t)(g * G + h) * HD + E * lane;
    float x[E];
    float peak = 0.f;
#pragma unroll
    for (int i = 0; i < E; ++i) x[i] = live ? q[i] : 0.f, peak = max_nan(peak, fabsf(x[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    const bool ok = peak < INFINITY;
    const int e = ok ? query_exp(peak) : 0;
    const Scale2 to_unit(-e);
    if (lane == 0) {
      s.unit[(int64_t)id * QB + r] = ok ? query_unit<HD>(e) : NAN;
      s.row_max[(int64_t)id * QB + r] = -INFINITY;
      s.own_max[(int64_t)id * QB + r] = -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float y0 = ok ? to_unit(x[i]) : 0.f, y1 = ok ? to_unit(x[i + 1]) : 0.f;
      const uint32_t hi = pack_half(y0, y1);
      const float2 f = __half22float2(*(const __half2*)&hi);
      uint8_t* p = dst + (r * HD + E * lane + i) * 2;
      *(uint32_t*)p = hi;
      *(uint32_t*)(p + QB * HD * 2) = pack_half(y0 - f.x, y1 - f.y);
    }
  }
}

// ---------------------------------------------------------------- the two passes
template <int HD, bool MAX>
struct TcSmem {
  static constexpr int TILE = 128 * HD * 2;  // bytes of a K or V tile
  // ring slots: as many as fit beside each other
  static constexpr int NK = (MAX ? 6 : 3) * (HD == 64 ? 2 : 1), NV = MAX ? 0 : NK;
  static constexpr int NS = MAX ? 3 : 2;     // score buffers (MAX has no O)
  static constexpr int K = 0, V = K + NK * TILE, SCALES = V + NV * TILE;
  static constexpr int BARS = SCALES + NSC * 2 * KB * 4;
  static constexpr size_t BYTES = (size_t)BARS + 512 + 1024;  // and alignment slack
};

// Ring position of a block: slot and the parity of its use
struct Ring {
  int slot = 0, parity = 0;
  template <int N>
  __device__ __forceinline__ void next() {
    if (++slot == N) slot = 0, parity ^= 1;
  }
};

// MAX: row maxima of the scores, and the V scales relative to their largest.  Else: the segments' O and weight sums.
template <int HD, bool MAX>
__global__ void __launch_bounds__(THREADS, 1) shared_pass_kernel(const __grid_constant__ SharedArgs s) {
  using M = TcSmem<HD, MAX>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint64_t* bar = (uint64_t*)(smem + M::BARS);
  uint64_t* q_full = bar;                // query rows are in TMEM
  uint64_t* s_full = bar + 1;            // [3] scores formed
  uint64_t* s_done = bar + 4;            // [3] MAX: scores read; else: P written
  uint64_t* pv_done = bar + 7;           // [2] P V formed: the score buffer is free
  uint64_t* sc_full = bar + 9;           // [NSC] scales are here
  uint64_t* sc_free = sc_full + NSC;     // [NSC]
  uint64_t* k_full = sc_free + NSC;      // [NK]
  uint64_t* k_free = k_full + M::NK;
  uint64_t* v_full = k_free + M::NK;     // [NV]
  uint64_t* v_free = v_full + M::NV;
  uint32_t* tmem_slot = (uint32_t*)(v_free + M::NV);
  const Kv8Attn& a = s.a;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int group = blockIdx.x / s.ways, way = blockIdx.x - group * s.ways;
  const int lines = s.tiles / s.ways;  // of a kv head
  const int u0 = group * s.per, u1 = min(s.units, u0 + s.per);

  if (tid == 0) {
    mbar_init(q_full, SOFT_WARPS);
    for (int i = 0; i < 3; ++i) mbar_init(&s_full[i], 1), mbar_init(&s_done[i], SOFT_WARPS);
    for (int i = 0; i < 2; ++i) mbar_init(&pv_done[i], 1);
    for (int i = 0; i < NSC; ++i) mbar_init(&sc_full[i], 1), mbar_init(&sc_free[i], SOFT_WARPS);
    for (int i = 0; i < 2 * (M::NK + M::NV); ++i) mbar_init(&k_full[i], 1);
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
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == LOAD_WARP) {
    if (lane == 0) {
      Ring k, v, sc;
      bool ok = true;
      for (int u = u0, j = 0; u < u1 && ok; ++u, ++j) {
        const int line = u / s.n_blocks;
        const int64_t from = (int64_t)(line / lines) * s.n_blocks + (u - line * s.n_blocks);
        if (j >= M::NK) ok = mbar_wait_bounded(&k_free[k.slot], k.parity ^ 1, a.status);
        if (!ok) break;
        mbar_expect_tx(&k_full[k.slot], M::TILE);
        bulk_g2s(smem + M::K + k.slot * M::TILE, s.kt + from * M::TILE, M::TILE, &k_full[k.slot]);
        k.next<M::NK>();
        if (j >= NSC) ok = mbar_wait_bounded(&sc_free[sc.slot], sc.parity ^ 1, a.status);
        if (!ok) break;
        mbar_expect_tx(&sc_full[sc.slot], 2 * KB * 4);
        bulk_g2s(smem + M::SCALES + sc.slot * (2 * KB * 4), s.scales + from * (2 * KB), 2 * KB * 4,
                 &sc_full[sc.slot]);
        sc.next<NSC>();
        if constexpr (!MAX) {
          if (j >= M::NV) ok = mbar_wait_bounded(&v_free[v.slot], v.parity ^ 1, a.status);
          if (!ok) break;
          mbar_expect_tx(&v_full[v.slot], M::TILE);
          bulk_g2s(smem + M::V + v.slot * M::TILE, s.vt + from * M::TILE, M::TILE, &v_full[v.slot]);
          v.next<M::NV>();
        }
      }
      // the tensor cores' last arrivals are in before the CTA's shared memory goes
      const int n = u1 - u0;
      for (int use = max(0, n - M::NK); use < n && ok; ++use) {
        ok = mbar_wait_bounded(&k_free[use % M::NK], use / M::NK & 1, a.status);
        if constexpr (!MAX) ok = ok && mbar_wait_bounded(&v_free[use % M::NV], use / M::NV & 1, a.status);
      }
    }
  } else if (warp == MMA_WARP) {
    const uint64_t kd0 = sw128_desc(smem_u32(smem + M::K)), vd0 = sw128_desc_mn(smem_u32(smem + M::V));
    bool ok = true;
    auto wait = [&](uint64_t* b, int parity) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait_bounded(b, parity, a.status));
    };
    Ring k, v, sb, pb;  // K and V slots; score buffers of the next scores and of the next P V
    int formed = 0;     // blocks whose scores have been started
    auto scores = [&]() {
      wait(&k_full[k.slot], k.parity);
      if (formed >= M::NS) wait(MAX ? &s_done[sb.slot] : &pv_done[sb.slot], sb.parity ^ 1);
      if (!ok) return;
      tc_fence_after();
      const uint64_t kd = kd0 + (uint32_t)(k.slot * (M::TILE >> 4));
      const uint32_t sd = tmem + TM_S + sb.slot * KB;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const uint64_t d = kd + (uint32_t)(((i >> 2) * (KB * 128) + (i & 3) * 32) >> 4);
        mma_ts(sd, tmem + TM_Q + 8 * i, d, idesc(KB, false), i != 0);
        mma_ts(sd, tmem + TM_Q + HD / 2 + 8 * i, d, idesc(KB, false), 1);
      }
      mma_commit(&s_full[sb.slot]);
      mma_commit(&k_free[k.slot]);
      k.next<M::NK>();
      sb.next<M::NS>();
      ++formed;
    };
    int seg = 0;
    for (int u = u0; u < u1 && ok; ++seg) {
      const int nb = min(u1 - u, s.n_blocks - u % s.n_blocks);
      wait(q_full, seg & 1);
      tc_fence_after();
      for (int i = 0; i < min(nb, M::NS) && ok; ++i) scores();
      for (int i = 0; i < nb && ok; ++i) {
        if constexpr (!MAX) {
          wait(&v_full[v.slot], v.parity);
          wait(&s_done[pb.slot], pb.parity);
          if (!ok) break;
          tc_fence_after();
          // keys 16 j ..: P hi, then lo, in the score columns of these keys
          const uint32_t p = tmem + TM_S + pb.slot * KB;
          const uint64_t vd = vd0 + (uint32_t)(v.slot * (M::TILE >> 4));
#pragma unroll
          for (int j = 0; j < KB / 16; ++j) {
            mma_ts(tmem + TM_O, p + 16 * j, vd + j * (16 * 128 >> 4), idesc(HD, true), i % FLUSH | j ? 1 : 0);
            mma_ts(tmem + TM_O, p + 16 * j + 8, vd + j * (16 * 128 >> 4), idesc(HD, true), 1);
          }
          mma_commit(&pv_done[pb.slot]);
          mma_commit(&v_free[v.slot]);
          v.next<M::NV>();
          pb.next<M::NS>();
        }
        if (i + M::NS < nb) scores();
      }
      u += nb;
    }
  } else {
    const int r = (warp & 3) * 32 + lane, part = warp >> 2;
    const uint32_t trow = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    __shared__ float red[PARTS][QB];
    bool ok = true;
    Ring sb, sc;
    // all lanes of a warp are done: one arrival
    auto arrive = [&](uint64_t* b) {
      __syncwarp();
      if (lane == 0) mbar_arrive(b);
    };
    // scores and scales of the next block are here
    auto enter = [&]() {
      ok = ok && mbar_wait_bounded(&sc_full[sc.slot], sc.parity, a.status);
      ok = ok && mbar_wait_bounded(&s_full[sb.slot], sb.parity, a.status);
      tc_fence_after();
    };
    if constexpr (MAX) {
      // this CTA's share of the V scales, relative to their head's largest (for the P V pass)
      const int n = a.c.n_kv * s.n_blocks, share = (n + gridDim.x - 1) / gridDim.x;
      for (int i = blockIdx.x * share + warp; i < min(n, ((int)blockIdx.x + 1) * share); i += SOFT_WARPS) {
        const int g = i / s.n_blocks;
        float m = 0x1p-126f;  // 1 / m is finite
        for (int e = lane; e < s.n_blocks * 4; e += 32) m = max_nan(m, s.v_max[(int64_t)g * s.n_blocks * 4 + e]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0 && i == g * s.n_blocks) s.v_top[g] = m;
        float4* v = (float4*)(s.scales + (int64_t)i * (2 * KB) + KB) + lane;
        float4 x = *v;
        const float mult = 1.f / m;
        x.x *= mult, x.y *= mult, x.z *= mult, x.w *= mult;
        *v = x;
      }
    }
    for (int u = u0; u < u1;) {
      const int line = u / s.n_blocks, g = line / lines, blk0 = u - line * s.n_blocks;
      const int tile = line * s.ways + way;  // of all kv heads
      const int nb = min(u1 - u, s.n_blocks - blk0);
      const int64_t row = (int64_t)tile * QB + r;
      {
        // this thread's part of its query row (hi | lo)
        constexpr int W = HD / PARTS;
        const uint4* q = (const uint4*)(s.qt + (int64_t)tile * (2 * QB * HD * 2) + r * (HD * 2));
#pragma unroll
        for (int i = 0; i < W; i += 16) {
          const int w = part * W + i;  // word of hi (HD / 2 of them), then of lo
          uint32_t x[16];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *(uint4*)&x[4 * e] = q[(w >= HD / 2 ? QB * HD * 2 / 16 + (w - HD / 2) / 4 : w / 4) + e];
          tmem_st16(trow + TM_Q + w, x);
        }
        tmem_wait_st();
        tc_fence_before();
        arrive(q_full);
      }
      if constexpr (MAX) {
        float m = -INFINITY;
        const Pair unit2(s.unit[row]);
        for (int i = 0; i < nb; ++i) {
          enter();
          const uint32_t k4 = smem_u32(smem + M::SCALES + sc.slot * (2 * KB * 4)) + part * (PK * 4);
          uint32_t x[PK / 32][32];
#pragma unroll
          for (int c = 0; c < PK / 32; ++c) tmem_ld32(trow + TM_S + sb.slot * KB + part * PK + 32 * c, x[c]);
#pragma unroll
          for (int c = 0; c < PK / 32; ++c) tmem_wait_ld(x[c]);
          tc_fence_before();
          arrive(&s_done[sb.slot]);
#pragma unroll
          for (int c = 0; c < PK / 32; ++c)
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 k = ld_slot(k4 + (32 * c + e) * 4);
              float y[4];
              mul2(Pair(__uint_as_float(x[c][e]), __uint_as_float(x[c][e + 1])), mul2(Pair(k.x, k.y), unit2))
                  .get(y[0], y[1]);
              mul2(Pair(__uint_as_float(x[c][e + 2]), __uint_as_float(x[c][e + 3])), mul2(Pair(k.z, k.w), unit2))
                  .get(y[2], y[3]);
              m = fmaxf(fmaxf(m, fmaxf(y[0], y[1])), fmaxf(y[2], y[3]));
            }
          arrive(&sc_free[sc.slot]);
          sb.next<M::NS>();
          sc.next<NSC>();
        }
        red[part][r] = m;
        soft_sync();
        if (part == 0) {
#pragma unroll
          for (int i = 1; i < PARTS; ++i) m = fmaxf(m, red[i][r]);
          atomic_max(s.row_max + row, m);
        }
        soft_sync();
      } else {
        // the row's maximum over the prefix and the own keys
        const float m = fmaxf(s.row_max[row], s.own_max[row]);
        const Pair unit2(s.unit[row]);
        Pair sum2(0.f);
        // weights of 16 keys, P over their scores; TAIL: only the first `left` keys exist
        auto weigh = [&](auto tail, uint32_t cols, const uint32_t (&x)[16], uint32_t k4, int left) {
          constexpr bool TAIL = decltype(tail)::value;
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 k = ld_slot(k4 + 4 * e), v = ld_slot(k4 + 4 * (KB + e));
#pragma unroll
            for (int o = 0; o < 2; ++o) {
              const Pair ku = mul2(o ? Pair(k.z, k.w) : Pair(k.x, k.y), unit2);
              // m is the largest of these rounded products, so the difference is 0 there and nowhere above: it must
              // not become one FMA with the product, as the packed add and multiply do (seen in their results)
              float z0, z1;
              mul2(Pair(__uint_as_float(x[e + 2 * o]), __uint_as_float(x[e + 2 * o + 1])), ku).get(z0, z1);
              Pair w = kv8_weight2(Pair(__fsub_rn(z0, m), __fsub_rn(z1, m)));
              if constexpr (TAIL) {
                float w0, w1;
                w.get(w0, w1);
                w = Pair(e + 2 * o < left ? w0 : 0.f, e + 2 * o + 1 < left ? w1 : 0.f);
              }
              sum2 = add2(sum2, w);
              const Pair p = mul2(w, o ? Pair(v.z, v.w) : Pair(v.x, v.y));
              float p0, p1;
              p.get(p0, p1);
              hi[e / 2 + o] = pack_half(p0, p1);
              const float2 f = __half22float2(*(const __half2*)&hi[e / 2 + o]);
              fma2(Pair(f.x, f.y), Pair(-1.f), p).get(p0, p1);
              lo[e / 2 + o] = pack_half(p0, p1);
            }
          }
          tmem_st8(cols, hi);
          tmem_st8(cols + 8, lo);
        };
        // O of the blocks since the last flush into the segment's sums, which this thread alone adds to
        const int64_t out = segment_of(s, group, line, way) * QB + r;
        const float vmax = s.v_top[g];
        bool stored = false;
        auto flush = [&](const Ring& pb) {
          ok = ok && mbar_wait_bounded(&pv_done[pb.slot], pb.parity, a.status);
          tc_fence_after();
          float4* o = (float4*)(s.acc + out * HD + part * (HD / PARTS));
#pragma unroll
          for (int c = 0; c < HD / PARTS / 16; ++c) {
            uint32_t x[16];
            tmem_ld16(trow + TM_O + part * (HD / PARTS) + 16 * c, x);
            tmem_wait_ld(x);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float4 y =
                  make_float4(__uint_as_float(x[4 * e]) * vmax, __uint_as_float(x[4 * e + 1]) * vmax,
                              __uint_as_float(x[4 * e + 2]) * vmax, __uint_as_float(x[4 * e + 3]) * vmax);
              if (stored)
                atomicAdd(o + 4 * c + e, y);
              else
                o[4 * c + e] = y;
            }
          }
          stored = true;
        };
        Ring last;  // the score buffer of the block before
        for (int i = 0; i < nb; ++i) {
          enter();
          const uint32_t k4 = smem_u32(smem + M::SCALES + sc.slot * (2 * KB * 4)) + part * (PK * 4);
          const uint32_t cols = trow + TM_S + sb.slot * KB + part * PK;
          const int left = a.prefix_len - (blk0 + i) * KB - part * PK;  // keys of this part that exist
          uint32_t x[PK / 16][16];
#pragma unroll
          for (int c = 0; c < PK / 16; ++c) tmem_ld16(cols + 16 * c, x[c]);
#pragma unroll
          for (int c = 0; c < PK / 16; ++c) tmem_wait_ld(x[c]);
          if (left >= PK) {
#pragma unroll
            for (int c = 0; c < PK / 16; ++c)
              weigh(std::false_type{}, cols + 16 * c, x[c], k4 + 64 * c, 0);
          } else {
#pragma unroll
            for (int c = 0; c < PK / 16; ++c)
              weigh(std::true_type{}, cols + 16 * c, x[c], k4 + 64 * c, left - 16 * c);
          }
          tmem_wait_st();
          if (i > 0 && i % FLUSH == 0) flush(last);  // before this block's P V starts O anew
          tc_fence_before();
          arrive(&s_done[sb.slot]);
          if (lane == 0) mbar_arrive(&sc_free[sc.slot]);
          last = sb;
          sb.next<M::NS>();
          sc.next<NSC>();
        }
        flush(last);
        float s0, s1;
        sum2.get(s0, s1);
        s0 += s1;
        red[part][r] = s0;
        soft_sync();
        if (part == 0) {
#pragma unroll
          for (int i = 1; i < PARTS; ++i) s0 += red[i][r];
          s.sum[out] = s0;
        }
        tc_fence_before();
        soft_sync();
      }
      u += nb;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
  }
}

// A thread: 4 dims of a row.  Grid: 256 threads, kv heads.
template <int HD>
__global__ void __launch_bounds__(256) shared_join_kernel(SharedArgs s) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;");
  const Kv8Attn& a = s.a;
  constexpr int L = HD / 4;
  const int row = blockIdx.x * (256 / L) + threadIdx.x / L, d = threadIdx.x % L * 4, g = blockIdx.y;
  if (row >= s.rows) return;
  const int G = a.n_heads / a.c.n_kv, b = row / G, h = row - b * G;
  int slot, len;
  if (!row_keys(a, b, slot, len)) return;
  const int tile = g * s.tiles + row / QB, r = row % QB;
  float4 x = {};
  float total = 0.f;
  auto add = [&](const float* acc, float sum) {
    const float4 y = *(const float4*)(acc + d);
    x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
    total += sum;
  };
  const int line = tile / s.ways, way = tile - line * s.ways;
#pragma unroll 4
  for (int c = line * s.n_blocks / s.per; c <= ((line + 1) * s.n_blocks - 1) / s.per; ++c) {
    const int64_t at = segment_of(s, c, line, way) * QB + r;
    add(s.acc + at * HD, s.sum[at]);
  }
  if (s.own_acc) {
    const int64_t at = (int64_t)tile * QB + r;
    add(s.own_acc + at * HD, s.own_sum[at]);
  }
  float* out = a.out + ((int64_t)b * a.n_heads + g * G + h) * HD + d;
  out[0] = __fdiv_rn(x.x, total), out[1] = __fdiv_rn(x.y, total);
  out[2] = __fdiv_rn(x.z, total), out[3] = __fdiv_rn(x.w, total);
}

template <int HD>
int launch_shared(const SharedArgs& s, const Kv8Own& own, float* own_space, int B, int sms, cudaStream_t st,
                  int* n_launch) {
  auto max_pass = shared_pass_kernel<HD, true>;
  auto pv_pass = shared_pass_kernel<HD, false>;
  constexpr size_t max_smem = TcSmem<HD, true>::BYTES, pv_smem = TcSmem<HD, false>::BYTES;
  SM_CUDA_TRY(cudaFuncSetAttribute(max_pass, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)max_smem));
  SM_CUDA_TRY(cudaFuncSetAttribute(pv_pass, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pv_smem));
  cudaLaunchAttribute attr[2];
  const int n_kv = s.a.c.n_kv;
  const int prep = 2 * n_kv * s.n_blocks + n_kv * s.tiles * (QB / 16);
  cudaLaunchConfig_t cfg = launch_config(dim3(prep), 256, 0, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, shared_prep_kernel<HD>, s));
  cfg = launch_config(dim3(s.n_ctas), THREADS, max_smem, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, max_pass, s));
  if (s.own_acc) SM_TRY(launch_kv8_own(own, own_space, HD, B, sms, st, n_launch));
  cfg = launch_config(dim3(s.n_ctas), THREADS, pv_smem, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, pv_pass, s));
  cfg = launch_config(dim3(ceil_div(s.rows, 1024 / HD), n_kv), 256, 0, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, shared_join_kernel<HD>, s));
  *n_launch += 4;
  return SM_OK;
}

}  // namespace

int launch_attention_shared_tc(const Kv8Attn& a, int hd, int B, int device, int sms, cudaStream_t st, int* n_launch) {
  SharedArgs s = {};
  s.a = a;
  const int n_kv = a.c.n_kv;
  const int64_t rows = (int64_t)B * (a.n_heads / n_kv);
  s.n_blocks = ceil_div(a.prefix_len, KB);
  s.tiles = ceil_div(rows, QB);
  s.rows = (int)rows;
  const int64_t tiles = (int64_t)n_kv * s.tiles, units = tiles * s.n_blocks;
  // unit, tile and grid indexes are 32-bit
  if (units > (1 << 30) || 2ll * n_kv * s.n_blocks + tiles * (QB / 16) > (1 << 30))
    return fail(SM_ERR_SHAPE, "attention_shared_kv8: batch times prefix too large");
  // as many ways as cost no more than 4 % in a CTA's blocks (256 rows over 32768 keys, sustained under the power
  // limit: 1, 2, 4, 8 ways 470, 451, 442, 439 us for the whole call)
  const int even = ceil_div(units, std::min<int64_t>(sms, units));
  for (s.ways = std::min(sms, s.tiles);; --s.ways) {
    if (s.tiles % s.ways) continue;
    s.units = (int)(units / s.ways);
    s.per = ceil_div(s.units, std::min(sms / s.ways, s.units));
    if (s.ways == 1 || s.per <= even * 1.04) break;
  }
  s.n_ctas = ceil_div(s.units, s.per) * s.ways;
  Kv8Own own = {};
  own.a = a;
  own.a.prefix_len = 0;
  if (a.max_len > 0) SM_TRY(plan_kv8_own(own, hd, B, device, sms));
  const int64_t tile = 128ll * hd * 2, rp = tiles * QB, segments = s.n_ctas + tiles;
  const int64_t blocks = (int64_t)n_kv * s.n_blocks;
  // every part in whole 16 bytes, the first ones in whole tiles
  const int64_t f_acc = segments * QB * hd, f_sum = segments * QB, f_scales = blocks * 2 * KB, f_vmax = blocks * 4,
                f_top = (n_kv + 3) & ~3, f_own = a.max_len > 0 ? rp * hd + rp + own.floats : 0;
  const int64_t bytes =
      (2 * blocks + 2 * tiles) * tile + (f_acc + f_sum + f_scales + 3 * rp + f_vmax + f_top + f_own) * 4;
  uint8_t* buf = nullptr;
  if (cudaMallocAsync((void**)&buf, (size_t)bytes, st) != cudaSuccess) {
    cudaGetLastError();
    return fail(SM_ERR_OOM, "attention_shared_kv8: device allocation failed");
  }
  s.kt = buf;
  s.vt = s.kt + blocks * tile;
  s.qt = s.vt + blocks * tile;
  s.acc = (float*)(s.qt + 2 * tiles * tile);
  s.sum = s.acc + f_acc;
  s.scales = s.sum + f_sum;
  s.unit = s.scales + f_scales;
  s.row_max = s.unit + rp;
  s.own_max = s.row_max + rp;
  s.v_max = s.own_max + rp;
  s.v_top = s.v_max + f_vmax;
  float* own_space = nullptr;
  if (f_own) {
    s.own_acc = s.v_top + f_top;
    s.own_sum = s.own_acc + rp * hd;
    own_space = s.own_sum + rp;
  }
  own.behind = {s.row_max, s.tiles * QB, s.own_max, s.own_acc, s.own_sum};
  const int rc = hd == 64 ? launch_shared<64>(s, own, own_space, B, sms, st, n_launch)
                          : launch_shared<128>(s, own, own_space, B, sms, st, n_launch);
  cudaFreeAsync(buf, st);
  return rc;
}

}  // namespace sm
