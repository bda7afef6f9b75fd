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

// Launch on a stream after its previous kernel by programmatic dependent launch: the kernel waits
// (griddepcontrol.wait) before it touches memory.  What it reads may thus be written while it already runs, so
// none of it goes through __restrict__ or the read-only path, whose loads may move ahead of the wait.  attr
// backs the result.
inline cudaLaunchConfig_t launch_config(dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster,
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

// One decode attention call.
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
  bool q_vec;  // rows of q on 16-byte boundaries
};

// Row b's slot and length; false where there is nothing to do (padding) or the row is out of range.
__device__ __forceinline__ bool row_keys(const Kv8Attn& a, int b, int& slot, int& len) {
  slot = a.seq_ids ? a.seq_ids[b] : b;
  if (slot < 0) return false;
  len = a.lens[b];
  if (slot >= a.c.slots || len < 0 || len > a.max_len) {
    if (threadIdx.x == 0) atomicExch(a.status, SM_ERR_SHAPE);
    return false;
  }
  return true;
}

// The same as a question
__device__ __forceinline__ bool row_in_range(const Kv8Attn& a, int b) {
  const int slot = a.seq_ids ? a.seq_ids[b] : b, len = a.lens[b];
  return slot >= 0 && slot < a.c.slots && len >= 0 && len <= a.max_len;
}

// For the own keys of a batch behind a shared prefix (attn_kv8_tc.cu), row = kv head * rows + b * group + head:
// what is known of the prefix's scores, and where the own part goes.
struct Kv8Behind {
  const float* prefix_max;  // largest score over the prefix; nullptr: there is no such prefix
  int rows;
  float* own_max;           // largest own score, -inf at first
  float* acc;               // [row][head_dim] sum of weights times values
  float* sum;               // [row] sum of weights
};

// Own-key attention behind a prefix: one launch or two; what they need beside the caller's arrays.
struct Kv8Own {
  Kv8Attn a;                 // prefix_len 0
  Kv8Behind behind;
  int cluster, cap, warps;   // the cluster form's size, keys and warps of a CTA; 0: the split form
  size_t smem;
  int64_t floats;            // the split form's workspace
};
int plan_kv8_own(Kv8Own& own, int head_dim, int B, int device, int sms);
int launch_kv8_own(const Kv8Own& own, float* workspace, int head_dim, int B, int sms, cudaStream_t st, int* n_launch);

// Larger of p and v into p, in any order of the calls; a NaN is dropped
__device__ __forceinline__ void atomic_max(float* p, float v) {
  v += 0.f;  // -0 as 0
  if (v >= 0.f)
    atomicMax((int*)p, __float_as_int(v));
  else if (v < 0.f)
    atomicMin((unsigned*)p, __float_as_uint(v));
}

// attn_kv8_tc.cu: decode attention behind a shared prefix (prefix_len > 0) on tcgen05
int launch_attention_shared_tc(const Kv8Attn& a, int head_dim, int B, int device, int sms, cudaStream_t st,
                               int* n_launch);

}  // namespace sm
