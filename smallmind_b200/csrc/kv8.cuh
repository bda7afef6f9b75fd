// The 8-bit KV cache: host checks shared by its entry points, and its addressing.
#pragma once
#include "common.cuh"

namespace sm {

// Checks a cache description on the host; `what` names the call.
int kv8_check(const sm_kv8* c, const char* what);

// What the kernels get of a cache (passed by value).
struct Kv8View {
  int8_t* k;
  int8_t* v;
  float* ks;
  float* vs;
  int slots, tokens, n_kv;
  // index of (slot, kv head, position) in the scale arrays; times head_dim in the code arrays
  __host__ __device__ int64_t at(int slot, int head, int pos) const {
    return ((int64_t)slot * n_kv + head) * tokens + pos;
  }
};

inline Kv8View kv8_view(const sm_kv8* c) {
  return {c->k, c->v, c->k_scale, c->v_scale, c->max_seqs, c->max_tokens, c->n_kv};
}

}  // namespace sm
