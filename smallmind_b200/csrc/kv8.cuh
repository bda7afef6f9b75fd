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

// The long form of the decode attention (attn_kv8.cu): scores of chunks of keys, then P V.  Also the own keys
// of the batch behind a shared prefix, whose maxima and sums then come from attn_kv8_tc.cu.
struct Kv8Split {
  Kv8Attn a;
  int chunk, n_chunks;  // keys of a chunk (whole blocks of 32); chunks that max_len makes
  int gp;               // heads a kv head's group is padded to: 4, 8 or 16
  float* z;             // [B][n_kv][gp / 8 or 1][blocks] blocks of scores
  float* pacc;          // [B][n_kv][n_chunks][gp][head_dim]
  float* stat;          // [B][n_kv][n_chunks][2 * gp + 1] maxima, largest V scale; then the weights' sums
  int* arrived;         // [B][n_kv] chunks whose P V is done
  // behind a shared prefix: the largest raw score of row b * group + head, [n_kv][prefix_rows], and its factor
  // (z = score * unit); the chunks are then joined by the caller
  const float* prefix_max;
  const float* prefix_unit;
  int prefix_rows;
};
// Sizes chunk, n_chunks and gp; returns the floats that z, pacc, stat and arrived take together.
int64_t kv8_split_plan(Kv8Split& s, int head_dim, int B, int sms);
void kv8_split_place(Kv8Split& s, int head_dim, int B, float* base);
int launch_kv8_split_scores(const Kv8Split& s, int head_dim, int B, cudaStream_t st);
int launch_kv8_split_pv(const Kv8Split& s, int head_dim, int B, cudaStream_t st);

// attn_kv8_tc.cu: decode attention behind a shared prefix (prefix_len > 0) on tcgen05
int launch_attention_shared_tc(const Kv8Attn& a, int head_dim, int B, int sms, cudaStream_t st, int* n_launch);

}  // namespace sm
