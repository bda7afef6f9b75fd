// Writing and reading the 8-bit KV cache.
//
// A head's row x[hd] is kept as codes c and one scale s:
//   s = fl32(max|x| * fl32(1 / 127)),  c = x / s rounded to the nearest integer (ties to even),
// and read back as fl32(c * s).  The rounding is exact: with q the candidate next to
// x * (1 / s), the remainder r = x - q * s is formed without error by one FMA (q has 7
// bits and |r| <= ~s, so r fits 24 bits), and q stands unless |r| >= s / 2.  That test
// fails only for values within an ulp or so of a border, which then take a float64
// division.  So the codes do not depend on how the quotient was formed.
//
// Both kernels are bound by HBM: a write moves 4 + 1 bytes a value and 4 a scale, a read
// the same.  A lane takes 4 neighbouring values (16 bytes of fp32, 4 of codes), a head's
// row sits in hd / 4 lanes of one warp, so the maximum is a few shuffles and every load
// and store of a warp is contiguous.
#include "kv8.cuh"

namespace sm {

int kv8_check(const sm_kv8* c, const char* what) {
  auto refuse = [&](int code, const char* why) { return fail(code, std::string(what) + ": " + why); };
  if (!c) return refuse(SM_ERR_INVALID_ARG, "null cache");
  if (c->max_seqs <= 0 || c->max_tokens <= 0 || c->n_kv <= 0) return refuse(SM_ERR_SHAPE, "bad cache shape");
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

// Slot and position of row i, or false where the row is padding or out of range.
__device__ __forceinline__ bool row_target(const int* seq_ids, const int* positions, int64_t i, const Kv8View& c,
                                           int* status, int& slot, int& pos) {
  slot = seq_ids[i];
  if (slot < 0) return false;
  pos = positions[i];
  if (slot >= c.slots || pos < 0 || pos >= c.tokens) {
    atomicExch(status, SM_ERR_SHAPE);
    return false;
  }
  return true;
}

__device__ __forceinline__ int code64(float x, float s) {
  const double q = rint((double)x / (double)s);
  return (int)fmin(fmax(q, -127.0), 127.0);
}

// Codes of four values under scale s, packed into a word (value 0 in the low byte).
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float s) {
  const float MAGIC = 12582912.f;  // 1.5 * 2^23: adding it leaves the rounded integer in the low mantissa bits
  const float inv = 1.f / s, half = 0.5f * s;
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

// Item (row, K | V, head), head fastest.  HD / 4 lanes an item.
template <int HD, bool VEC>
__global__ void __launch_bounds__(THREADS) kv8_write_kernel(Kv8View c, const float* __restrict__ k,
                                                            const float* __restrict__ v, int64_t row_stride,
                                                            const int* __restrict__ seq_ids,
                                                            const int* __restrict__ positions, int64_t n_items,
                                                            int* status) {
  constexpr int LANES = HD / 4;
  const int lane = threadIdx.x % LANES;
  const int64_t item = (int64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
  int slot = 0, pos = 0, head = 0;
  bool is_v = false, live = false;
  float x[4] = {0.f, 0.f, 0.f, 0.f};
  if (item < n_items) {
    const int64_t row = item / (2 * c.n_kv);
    head = (int)(item - row * (2 * c.n_kv));
    is_v = head >= c.n_kv;
    if (is_v) head -= c.n_kv;
    live = row_target(seq_ids, positions, row, c, status, slot, pos);
    if (live) {
      const float* src = (is_v ? v : k) + row * row_stride + head * HD + 4 * lane;
      if (VEC) {
        const float4 t = *(const float4*)src;
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = src[i];
      }
    }
  }
  // the maximum as bits: non-negative floats order like integers, and infinities and NaNs lie above them
  int peak = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) peak = max(peak, __float_as_int(x[i]) & 0x7fffffff);
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, o));
  if (!live) return;
  uint32_t word = 0;
  float s = __int_as_float(peak) * (1.f / 127.f);
  if (peak >= 0x7f800000)
    s = __int_as_float(0x7fffffff);
  else if (s > 0.f)
    word = codes4(x, s);
  const int64_t at = c.at(slot, head, pos);
  *(uint32_t*)((is_v ? c.v : c.k) + at * HD + 4 * lane) = word;
  if (lane == 0) (is_v ? c.vs : c.ks)[at] = s;
}

template <int HD, bool VEC>
__global__ void __launch_bounds__(THREADS) kv8_read_kernel(Kv8View c, const int* __restrict__ seq_ids,
                                                           const int* __restrict__ positions, int64_t n_items,
                                                           float* __restrict__ k, float* __restrict__ v,
                                                           int64_t row_stride, int* status) {
  constexpr int LANES = HD / 4;
  const int lane = threadIdx.x % LANES;
  const int64_t item = (int64_t)blockIdx.x * (THREADS / LANES) + threadIdx.x / LANES;
  if (item >= n_items) return;
  const int64_t row = item / (2 * c.n_kv);
  int head = (int)(item - row * (2 * c.n_kv));
  const bool is_v = head >= c.n_kv;
  if (is_v) head -= c.n_kv;
  float* to = is_v ? v : k;
  int slot, pos;
  if (!to || !row_target(seq_ids, positions, row, c, status, slot, pos)) return;
  const int64_t at = c.at(slot, head, pos);
  const char4 w = *(const char4*)((is_v ? c.v : c.k) + at * HD + 4 * lane);
  const float s = (is_v ? c.vs : c.ks)[at];
  to += row * row_stride + head * HD + 4 * lane;
  const float4 y = make_float4((float)w.x * s, (float)w.y * s, (float)w.z * s, (float)w.w * s);
  if (VEC) {
    *(float4*)to = y;
  } else {
    to[0] = y.x, to[1] = y.y, to[2] = y.z, to[3] = y.w;
  }
}

int check_rows(sm_ctx* ctx, const sm_kv8* c, const int* seq_ids, const int* positions, int n_rows, int64_t row_stride,
               const char* what) {
  auto refuse = [&](int code, const char* why) { return fail(code, std::string(what) + ": " + why); };
  SM_TRY(kv8_check(c, what));
  if (n_rows < 0) return refuse(SM_ERR_SHAPE, "n_rows must not be negative");
  if (row_stride < (int64_t)c->n_kv * c->head_dim) return refuse(SM_ERR_SHAPE, "row_stride is less than a row");
  if (!ctx || (n_rows && (!seq_ids || !positions))) return refuse(SM_ERR_INVALID_ARG, "null argument");
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
  SM_TRY(check_rows(ctx, cache, seq_ids, positions, n_rows, row_stride, "kv8_write"));
  if (n_rows == 0) return SM_OK;
  if (!k || !v) return fail(SM_ERR_INVALID_ARG, "kv8_write: null argument");
  int device = 0;
  cudaStream_t st = nullptr;
  int64_t* launches = nullptr;
  SM_TRY(ctx_view(ctx, &device, &st, &launches));
  DeviceGuard guard(device);
  const Kv8View c = kv8_view(cache);
  const int64_t items = (int64_t)n_rows * 2 * c.n_kv;
  const int64_t grid = (items * (cache->head_dim / 4) + THREADS - 1) / THREADS;
  if (grid > INT32_MAX) return fail(SM_ERR_SHAPE, "kv8_write: too many rows");
  const bool vec = rows_vectorizable(k, v, row_stride);
  auto kern = cache->head_dim == 64 ? (vec ? kv8_write_kernel<64, true> : kv8_write_kernel<64, false>)
                                    : (vec ? kv8_write_kernel<128, true> : kv8_write_kernel<128, false>);
  kern<<<(int)grid, THREADS, 0, st>>>(c, k, v, row_stride, seq_ids, positions, items, ctx_status(ctx));
  SM_CUDA_TRY(cudaGetLastError());
  *launches += 1;
  return SM_OK;
}

SM_API int sm_kv8_read(sm_ctx* ctx, const sm_kv8* cache, const int* seq_ids, const int* positions, int n_rows,
                       float* k, float* v, int64_t row_stride) {
  SM_TRY(check_rows(ctx, cache, seq_ids, positions, n_rows, row_stride, "kv8_read"));
  if (n_rows == 0) return SM_OK;
  if (!k && !v) return fail(SM_ERR_INVALID_ARG, "kv8_read: null argument");
  int device = 0;
  cudaStream_t st = nullptr;
  int64_t* launches = nullptr;
  SM_TRY(ctx_view(ctx, &device, &st, &launches));
  DeviceGuard guard(device);
  const Kv8View c = kv8_view(cache);
  const int64_t items = (int64_t)n_rows * 2 * c.n_kv;
  const int64_t grid = (items * (cache->head_dim / 4) + THREADS - 1) / THREADS;
  if (grid > INT32_MAX) return fail(SM_ERR_SHAPE, "kv8_read: too many rows");
  const bool vec = rows_vectorizable(k, v, row_stride);
  auto kern = cache->head_dim == 64 ? (vec ? kv8_read_kernel<64, true> : kv8_read_kernel<64, false>)
                                    : (vec ? kv8_read_kernel<128, true> : kv8_read_kernel<128, false>);
  kern<<<(int)grid, THREADS, 0, st>>>(c, seq_ids, positions, items, k, v, row_stride, ctx_status(ctx));
  SM_CUDA_TRY(cudaGetLastError());
  *launches += 1;
  return SM_OK;
}

}  // extern "C"
