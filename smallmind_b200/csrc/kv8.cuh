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
// (griddepcontrol.wait) before it touches memory.  attr backs the result.
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

}  // namespace sm
