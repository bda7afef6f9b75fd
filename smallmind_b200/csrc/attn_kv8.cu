// Decode attention over the 8-bit KV cache, with and without a prefix shared by the batch.
//
// Row (b, h) with keys j (the shared prefix's first, then the sequence's own):
//   z_j = (q . k_j) / sqrt(hd),  m = max_j z_j,  x_j = max(z_j - m, -87.3),
//   e_j = (12 + 6 x_j + x_j^2) / (12 - 6 x_j + x_j^2),  out = sum_j e_j v_j / sum_j e_j.
// e is the reference's rational FastExp (MathUtils.cs:20-32).  It is not multiplicative, so
// partial results against a running maximum cannot be rescaled: the exact maximum comes
// first and the weights are formed against it.
#include "kv8.cuh"

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

// x <= 0 or NaN, which has to come out as NaN
__device__ __forceinline__ float weight(float x) {
  x = x < -87.3f ? -87.3f : x;
  const float a = fmaf(x, x, 12.f);
  return __fdividef(fmaf(6.f, x, a), fmaf(-6.f, x, a));
}

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
    if ((int)threadIdx.x < n) es[threadIdx.x] = weight(score(j0 + threadIdx.x) - m);
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

int attend(sm_ctx* ctx, const Kv8Attn& args, int head_dim, int B, const char* what) {
  int device = 0;
  cudaStream_t st = nullptr;
  int64_t* launches = nullptr;
  SM_TRY(ctx_view(ctx, &device, &st, &launches));
  DeviceGuard guard(device);
  Kv8Attn a = args;
  a.status = ctx_status(ctx);
  const dim3 grid(a.n_heads, B);
  if (B > 65535) return fail(SM_ERR_SHAPE, std::string(what) + ": batch too large");
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
