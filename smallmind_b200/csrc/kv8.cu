// Writing and reading the 8-bit KV cache.
//
// A head's row x[hd] is kept as codes c and one scale s:
//   s = fl32(max|x| * fl32(1 / 127)),  c = x / s rounded to the nearest integer (ties to even),
// and read back as fl32(c * s).  The scale is a product, within two ulps of the quotient max|x| / 127, because that
// is what torch makes of x / 127.0 on the GPU (equal on 4 M values): rows quantised there and here have the same
// scales and codes.  The rounding of the codes is exact: with q the candidate next to
// x * (1 / s), the remainder r = x - q * s is formed without error by one FMA (q has 7
// bits and |r| <= ~s, so r fits 24 bits), and q stands unless |r| >= s / 2.  That test
// fails only for values within an ulp or so of a border, which then take a float64
// division.  So the codes do not depend on how the quotient was formed.
//
// Both kernels are bound by HBM: a write moves 4 + 1 bytes a value and 4 a scale, a read the same.  A lane
// takes 4 neighbouring values (16 bytes of fp32, 4 of codes), so every access of a warp is contiguous and a
// head's maximum is one reduction over its 16 or 32 lanes.  What hides the latency is bytes on their way: a
// warp takes several pieces of 128 values and starts all of their loads before it uses the first.  (32768 rows of 8
// heads of 128, written and read back: 111 us, floor 94 us; 65536 rows read: 111 us, floor 104 us.)
#include <algorithm>

#include "kv8.cuh"

namespace sm {

int kv8_check(const sm_kv8* c, const char* what) {
  auto refuse = [&](int code, const char* why) { return fail(code, std::string(what) + ": " + why); };
  if (!c) return refuse(SM_ERR_INVALID_ARG, "null cache");
  if (c->max_seqs <= 0 || c->max_tokens <= 0 || c->n_kv <= 0) return refuse(SM_ERR_SHAPE, "bad cache shape");
  if (c->n_kv > 4096) return refuse(SM_ERR_UNSUPPORTED, "more than 4096 kv heads");
  if (c->head_dim != 64 && c->head_dim != 128) return refuse(SM_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return refuse(SM_ERR_INVALID_ARG, "null cache array");
  if (((uintptr_t)c->k | (uintptr_t)c->v) % 16)
    return refuse(SM_ERR_INVALID_ARG, "the code arrays must be 16-byte aligned");
  if (((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 4)
    return refuse(SM_ERR_INVALID_ARG, "the scale arrays must be 4-byte aligned");
  return SM_OK;
}

namespace {

constexpr int THREADS = 256;

// The kernels are launched before the one ahead of them on the stream has ended and wait for it themselves, so
// what they read may still be written while they run: no __restrict__, no read-only loads.

// Whether a row is neither padding nor out of range
__device__ __forceinline__ bool in_cache(const Kv8View& c, int slot, int pos, int* status) {
  if (slot < 0) return false;
  if (slot < c.slots && pos >= 0 && pos < c.tokens) return true;
  atomicExch(status, SM_ERR_SHAPE);
  return false;
}

__device__ __forceinline__ int code64(float x, float s) {
  const double q = rint((double)x / (double)s);
  return (int)fmin(fmax(q, -127.0), 127.0);
}

// Codes of four values under scale s, packed into a word (value 0 in the low byte).
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float s) {
  const float MAGIC = 12582912.f;  // 1.5 * 2^23: adding it leaves the rounded integer in the low mantissa bits
  const float inv = __fdividef(1.f, s), half = 0.5f * s;  // an approximate quotient: the remainder decides
  uint32_t bits[4];
  bool near_border = s < 1e-30f;  // where s / 2 or 1 / s might round
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float t = fmaf(x[i], inv, MAGIC);
    const float r = fmaf(-(t - MAGIC), s, x[i]);
    near_border |= fabsf(r) >= half;
    bits[i] = __float_as_uint(t);
  }
  if (near_border) {
#pragma unroll
    for (int i = 0; i < 4; ++i) bits[i] = (uint32_t)code64(x[i], s);
  }
  return __byte_perm(__byte_perm(bits[0], bits[1], 0x0040), __byte_perm(bits[2], bits[3], 0x0040), 0x5410);
}

// A warp's share of a write: N pieces of 128 values, from piece N * (blockIdx.y / 2), of the K (even blockIdx.y) or V
// values of row blockIdx.x * warps + warp.  Both sides are walked by constant steps.  Rows run fastest, so
// CTAs that run together touch few heads (the other order: 8 to 13 % slower).
template <int HD, int N>
struct Share {
  int row, value, dim, left;  // row; this lane's first value in it; its dim; values from it to the row's end
  int64_t step;               // from a piece's place in the cache to the next one's, in positions
  bool is_v;
  __device__ __forceinline__ Share(const Kv8View& c) {
    const int lane = threadIdx.x % 32;
    row = blockIdx.x * (THREADS / 32) + threadIdx.x / 32;
    is_v = blockIdx.y & 1;
    value = (int)(blockIdx.y >> 1) * (N * 128) + 4 * lane;
    dim = value % HD;
    left = c.n_kv * HD - value;
    step = (int64_t)c.tokens * (128 / HD);
  }
  // this lane's place in the cache: position and head of its first value
  __device__ __forceinline__ int64_t at(const Kv8View& c, int slot, int pos) const {
    return c.at(slot, value / HD, pos);
  }
};

// CTAs of the write kernel an SM: what its registers allow.  The grid holds so many, and a warp starts the loads of
// its next row before it quantises the one that has come (32768 rows of 8 heads of 128, written and read back: 12 us
// less than with a warp for every row; 2, 4, 6 CTAs an SM 16, 15, 2 us more than 3; with 1, 2, 8 pieces 20, 4,
// 2 us more than with 4; 4 rows of one piece through shared memory, as in the read, 7 us more).
constexpr int write_ctas(int n) { return n == 4 ? 3 : 4; }

template <int HD, int N, bool VEC>
__global__ void __launch_bounds__(THREADS, write_ctas(N))
    kv8_write_kernel(Kv8View c, const float* k, const float* v, int64_t row_stride, const int* seq_ids,
                     const int* positions, int n_rows, int* status) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Share<HD, N> w(c);
  const int step = gridDim.x * (THREADS / 32);
  const float* src = (w.is_v ? v : k) + w.value;
  float x[N][4];
  int slot = -1, pos = 0;
  // the values do not wait for the ids to be checked (3 % slower)
  auto load = [&](int64_t row) {
    if (row >= n_rows) return;
    slot = seq_ids[row], pos = positions[row];
    const float* from = src + row * row_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
      if (w.left > i * 128) {
        if (VEC) {
          *(float4*)x[i] = __ldcs((const float4*)(from + i * 128));
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[i][e] = from[i * 128 + e];
        }
      }
    }
  };
  load(w.row);
  for (int64_t row = w.row; row < n_rows; row += step) {
    float y[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) y[i][e] = x[i][e];
    const int to_slot = slot, to_pos = pos;
    load(row + step);
    if (!in_cache(c, to_slot, to_pos, status)) continue;
    const int64_t at = w.at(c, to_slot, to_pos);
    int8_t* codes = (w.is_v ? c.v : c.k) + at * HD + w.dim;
    float* scales = (w.is_v ? c.vs : c.ks) + at;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // the maximum as bits: non-negative floats order like integers, and infinities and NaNs lie above them
      unsigned peak = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) peak = max(peak, __float_as_uint(y[i][e]) & 0x7fffffffu);
      peak = __reduce_max_sync(HD == 128 ? 0xffffffffu : threadIdx.x % 32 < 16 ? 0xffffu : 0xffff0000u, peak);
      if (w.left > i * 128) {
        uint32_t word = 0;
        float s = __uint_as_float(peak) * (1.f / 127.f);
        if (peak >= 0x7f800000u)
          s = __uint_as_float(0x7fffffffu);
        else if (s > 0.f)
          word = codes4(y[i], s);
        *(uint32_t*)codes = word;
        if (w.dim == 0) *scales = s;
      }
      codes += w.step * HD;
      scales += w.step;
    }
  }
}

// N pieces of 128 K or V values as above, of 4 rows a warp: a lane reads 16 neighbouring codes of one of them, so
// that there are enough bytes on their way, and they pass through shared memory to come out as one row after the
// other, 4 values a lane (65536 rows of 8 heads of 128: 112 us; 128 us with one row a warp, a lane reading the 4
// codes that it writes).
template <int HD, int N, bool VEC>
__global__ void __launch_bounds__(THREADS) kv8_read_kernel(Kv8View c, const int* seq_ids, const int* positions,
                                                           int n_rows, float* k, float* v, int64_t row_stride,
                                                           int* status) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ int4 words[THREADS / 32][N][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t row0 = 4 * ((int64_t)blockIdx.x * (THREADS / 32) + warp), row = row0 + lane / 8;
  const bool is_v = blockIdx.y & 1;
  const int piece = (int)(blockIdx.y >> 1) * N, values = c.n_kv * HD;
  float* to = is_v ? v : k;
  if (row0 >= n_rows || !to) return;
  int slot = -1, pos = 0;
  if (row < n_rows) slot = seq_ids[row], pos = positions[row];
  const bool live = in_cache(c, slot, pos, status);
  const unsigned rows = __ballot_sync(0xffffffffu, live);
  float s[N];
  int4 q[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int value = (piece + i) * 128 + lane % 8 * 16;
    s[i] = 0.f;
    q[i] = make_int4(0, 0, 0, 0);
    if (live && value < values) {
      const int64_t at = c.at(slot, value / HD, pos);
      q[i] = *(const int4*)((is_v ? c.v : c.k) + at * HD + value % HD);
      s[i] = (is_v ? c.vs : c.ks)[at];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i) words[warp][i][lane] = q[i];
  __syncwarp();
  to += row0 * row_stride + piece * 128 + 4 * lane;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const char4 x = ((const char4*)words[warp][i])[r * 32 + lane];
      const float f = __shfl_sync(0xffffffffu, s[i], r * 8 + lane / 4);
      if (!(rows >> (8 * r) & 1) || (piece + i) * 128 + 4 * lane >= values) continue;
      float* out = to + r * row_stride + i * 128;
      const float4 y = make_float4((float)x.x * f, (float)x.y * f, (float)x.z * f, (float)x.w * f);
      if (VEC) {
        __stcs((float4*)out, y);
      } else {
        out[0] = y.x, out[1] = y.y, out[2] = y.z, out[3] = y.w;
      }
    }
}

int check_rows(sm_ctx* ctx, const sm_kv8* c, const int* seq_ids, const int* positions, int n_rows, int64_t row_stride,
               const float* k, const float* v, const char* what) {
  auto refuse = [&](int code, const char* why) { return fail(code, std::string(what) + ": " + why); };
  SM_TRY(kv8_check(c, what));
  if (n_rows < 0) return refuse(SM_ERR_SHAPE, "n_rows must not be negative");
  if (row_stride < (int64_t)c->n_kv * c->head_dim) return refuse(SM_ERR_SHAPE, "row_stride is less than a row");
  if (!ctx || (n_rows && (!seq_ids || !positions))) return refuse(SM_ERR_INVALID_ARG, "null argument");
  if (((uintptr_t)k | (uintptr_t)v | (uintptr_t)seq_ids | (uintptr_t)positions) % 4)
    return refuse(SM_ERR_INVALID_ARG, "misaligned pointer");
  return SM_OK;
}

bool rows_vectorizable(const float* a, const float* b, int64_t row_stride) {
  return ((uintptr_t)a | (uintptr_t)b) % 16 == 0 && row_stride % 4 == 0;
}

}  // namespace
}  // namespace sm

using namespace sm;

extern "C" {

SM_API int sm_kv8_write(sm_ctx* ctx, const sm_kv8* cache, const float* k, const float* v, int64_t row_stride,
                        const int* seq_ids, const int* positions, int n_rows) {
  SM_TRY(check_rows(ctx, cache, seq_ids, positions, n_rows, row_stride, k, v, "kv8_write"));
  if (n_rows == 0) return SM_OK;
  if (!k || !v) return fail(SM_ERR_INVALID_ARG, "kv8_write: null argument");
  int device = 0;
  cudaStream_t st = nullptr;
  int64_t* launches = nullptr;
  SM_TRY(ctx_view(ctx, &device, &st, &launches));
  DeviceGuard guard(device);
  const Kv8View c = kv8_view(cache);
  const int pieces = ceil_div((int64_t)c.n_kv * cache->head_dim, 128), n = pieces >= 3 ? 4 : pieces;
  const int parts = 2 * ceil_div(pieces, n);
  int sms = 0;
  SM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  const dim3 grid(std::min(ceil_div(n_rows, THREADS / 32), std::max(1, write_ctas(n) * sms / parts)), parts);
  const bool vec = rows_vectorizable(k, v, row_stride);
  const int which = (cache->head_dim == 64 ? 0 : 6) + (n == 4 ? 4 : 2 * (n - 1)) + vec;
  decltype(&kv8_write_kernel<64, 1, false>) const kernels[] = {
      kv8_write_kernel<64, 1, false>,  kv8_write_kernel<64, 1, true>,  kv8_write_kernel<64, 2, false>,
      kv8_write_kernel<64, 2, true>,   kv8_write_kernel<64, 4, false>, kv8_write_kernel<64, 4, true>,
      kv8_write_kernel<128, 1, false>, kv8_write_kernel<128, 1, true>, kv8_write_kernel<128, 2, false>,
      kv8_write_kernel<128, 2, true>,  kv8_write_kernel<128, 4, false>, kv8_write_kernel<128, 4, true>};
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = launch_config(grid, THREADS, 0, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernels[which], c, k, v, row_stride, seq_ids, positions, n_rows,
                                 ctx_status(ctx)));
  *launches += 1;
  return SM_OK;
}

SM_API int sm_kv8_read(sm_ctx* ctx, const sm_kv8* cache, const int* seq_ids, const int* positions, int n_rows,
                       float* k, float* v, int64_t row_stride) {
  SM_TRY(check_rows(ctx, cache, seq_ids, positions, n_rows, row_stride, k, v, "kv8_read"));
  if (n_rows == 0) return SM_OK;
  if (!k && !v) return fail(SM_ERR_INVALID_ARG, "kv8_read: null argument");
  int device = 0;
  cudaStream_t st = nullptr;
  int64_t* launches = nullptr;
  SM_TRY(ctx_view(ctx, &device, &st, &launches));
  DeviceGuard guard(device);
  const Kv8View c = kv8_view(cache);
  const int pieces = ceil_div((int64_t)c.n_kv * cache->head_dim, 128), groups = ceil_div(n_rows, 4 * (THREADS / 32));
  int sms = 0;
  SM_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
  // two pieces a warp once that leaves 32 CTAs an SM (2500 rows of 8 heads of 128: 1 piece 4.6 us, 2 pieces 6.0 us;
  // 65536 rows: 115 and 112 us)
  const int n = (int64_t)groups * pieces >= 32ll * sms ? 2 : 1;
  const dim3 grid(groups, 2 * ceil_div(pieces, n));
  const bool vec = rows_vectorizable(k, v, row_stride);
  const int which = (cache->head_dim == 64 ? 0 : 4) + 2 * (n - 1) + vec;
  decltype(&kv8_read_kernel<64, 1, false>) const kernels[] = {
      kv8_read_kernel<64, 1, false>,  kv8_read_kernel<64, 1, true>,  kv8_read_kernel<64, 2, false>,
      kv8_read_kernel<64, 2, true>,   kv8_read_kernel<128, 1, false>, kv8_read_kernel<128, 1, true>,
      kv8_read_kernel<128, 2, false>, kv8_read_kernel<128, 2, true>};
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t cfg = launch_config(grid, THREADS, 0, st, 1, attr);
  SM_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernels[which], c, seq_ids, positions, n_rows, k, v, row_stride,
                                 ctx_status(ctx)));
  *launches += 1;
  return SM_OK;
}

}  // extern "C"
