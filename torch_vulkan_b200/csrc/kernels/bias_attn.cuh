// Attention with a learned relative position bias: parameters and device helpers shared by the SIMT and the
// tensor-core kernels.
//
//   x_ij = scale q_i.k_j + table[bucket(j - i - q_offset)][h]      keys j masked by key_mask, and j > i + q_offset
//   P = softmax_j(x), O = P V                                      when causal
//   dP = dO V^T, delta_i = sum_d dO O, dS = P (dP - delta), dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO,
//   dtable[n][h] = sum of dS over batch and over the pairs whose bucket is n
//
// The bias depends on j - i alone and is constant beyond +-max_distance, so a kernel holds it as one vector per head
// in shared memory. Everything is kept in units of log2 (x * log2 e) so that the exponential is one exp2.
#pragma once

#include "common.cuh"

namespace b2 {
namespace bias_attn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* o32;           // unrounded O [B*H*Sq][D], NULL: not kept
  float* lse;
  const float* table;
  const uint8_t* mask;
  const void* d_o;
  void* dq;
  void* dk;
  void* dv;
  const float* delta;   // [B*H*Sq] rowsum(dO * O)
  uint32_t* norms;      // [B*Hk][2] bits of the largest squared norms of a dO row and of a V row, f16 on the tensor cores
  float* dtab;          // [B*H][query tiles][num_buckets] partial sums, NULL: not wanted
  float* part_o;        // [nsplit][B*H*Sq][D] unnormalised outputs of the key splits
  float2* part_ml;      // [nsplit][B*H*Sq] (running maximum in log2 units, sum)
  int64_t q_s[3], k_s[3], v_s[3], o_s[3], do_s[3], dq_s[3], dk_s[3], dv_s[3];
  int64_t mask_sb;
  int B, H, Hk, Sq, Sk, D;
  int q_off;
  int R;                // max_distance
  int nb;               // num_buckets
  int bidir, causal;
  int nsplit;           // key splits of the forward (grid.z)
  int nthr;
  uint16_t thr[B2_BIAS_MAX_BUCKETS];  // bucket of a one-sided distance n = number of thresholds <= n
  float scale;
  int* err;
};

// Bucket of the relative position rel (|rel| <= R).
__device__ __forceinline__ int bucket_of(const Params& p, int rel) {
  const int n = p.bidir ? abs(rel) : max(-rel, 0);
  int c = 0;
  for (int i = 0; i < p.nthr; ++i) c += (n >= (int)p.thr[i]) ? 1 : 0;
  return c + (p.bidir && rel > 0 ? p.nb / 2 : 0);
}

// Bias of head h at a relative position, in log2 units; -inf where the causal mask hides the key.
__device__ __forceinline__ float bias_at(const Params& p, int h, int rel) {
  if (p.causal && rel > 0) return -INFINITY;
  const int r = max(-p.R, min(p.R, rel));
  return p.table[(int64_t)bucket_of(p, r) * p.H + h] * kLog2e;
}

// What a row's unnormalised output is multiplied by, and its log-sum, from the running maximum m (log2 units) and sum l. A sum of
// zero is a row without a key: zeros, and a log-sum of -inf. A NaN sum (a NaN or infinite score) stays one.
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.f / l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }

template <typename T>
__device__ __forceinline__ const T* row_of(const void* base, const int64_t* s, int b, int h, int64_t i) {
  return (const T*)base + b * s[0] + h * s[1] + i * s[2];
}
template <typename T>
__device__ __forceinline__ T* row_of(void* base, const int64_t* s, int b, int h, int64_t i) {
  return (T*)base + b * s[0] + h * s[1] + i * s[2];
}

// First key past the last one that query row i may see.
__device__ __forceinline__ int key_end(const Params& p, int64_t last_row) {
  if (!p.causal) return p.Sk;
  const int64_t e = last_row + p.q_off + 1;
  return e < 0 ? 0 : (e < p.Sk ? (int)e : p.Sk);
}

// What the mask leaves of the keys below `end`: one past the last, how many up to key lo and from key hi on, and the first two
// (INT_MAX: there is none). Every thread of the block calls it and gets the same; the row of the mask is read at
// once, in one trip to memory. slot: five ints of shared memory per warp, free again after the block's next barrier.
struct Visible {
  int last, past, ahead, first, second;
};
__device__ __forceinline__ Visible visible_keys(const Params& p, int b, int end, int lo, int hi, int nthreads, int* slot) {
  constexpr int NONE = 0x7fffffff;
  if (p.mask == nullptr)
    return {end, max(0, min(end, lo + 1)), max(0, end - max(0, hi)), end > 0 ? 0 : NONE, end > 1 ? 1 : NONE};
  const uint8_t* m = p.mask + (int64_t)b * p.mask_sb;
  Visible v = {0, 0, 0, NONE, NONE};
#pragma unroll 8
  for (int j = (int)threadIdx.x; j < end; j += nthreads) {
    const bool on = m[j] != 0;
    v.last = on ? j + 1 : v.last;
    v.past += on && j <= lo, v.ahead += on && j >= hi;
    v.second = on ? min(v.second, max(v.first, j)) : v.second;
    v.first = on ? min(v.first, j) : v.first;
  }
  // the lanes' into one, then the warps', which every warp joins for itself
  auto join = [](Visible a, bool counts) -> Visible {
    const unsigned all = 0xffffffffu;
    const int first = __reduce_min_sync(all, a.first);
    return {__reduce_max_sync(all, a.last), __reduce_add_sync(all, counts ? a.past : 0),
            __reduce_add_sync(all, counts ? a.ahead : 0), first, __reduce_min_sync(all, a.first == first ? a.second : a.first)};
  };
  v = join(v, true);
  const int lane = threadIdx.x & 31, warps = nthreads / 32;
  if (lane == 0) {
    int* s = slot + (threadIdx.x >> 5) * 5;
    s[0] = v.last, s[1] = v.past, s[2] = v.ahead, s[3] = v.first, s[4] = v.second;
  }
  __syncthreads();
  const int* s = slot + min(lane, warps - 1) * 5;
  return join(Visible{s[0], s[1], s[2], s[3], s[4]}, lane < warps);
}
// Whether query row i sees exactly one key. P is 1 there whatever the score, so dS is zero.
__device__ __forceinline__ bool sees_one(const Params& p, int i, int first, int second) {
  const int lim = p.causal ? i + p.q_off : p.Sk - 1;
  return first <= lim && second > lim;
}

int simt_fwd(const Params& p, int dtype, cudaStream_t st);   // bias_attn_simt.cu
int simt_bwd(const Params& p, int dtype, cudaStream_t st);
constexpr int kSimtTile = 32, kSimtWalk = 64;
bool tc_fwd_eligible(const b2_bias_attn_args* a);            // bias_attn_tc.cu
bool tc_bwd_eligible(const b2_bias_attn_args* a);
int tc_fwd(const Params& p, bool bf16, cudaStream_t st);
int tc_bwd(const Params& p, bool bf16, float2* lsed, int sq_pad, cudaStream_t st);
constexpr int kTcTile = 128;
bool rows_eligible(const b2_bias_attn_args* a);              // bias_attn_rows.cu
int rows_blocks_per_sm(const b2_bias_attn_args* a);
int rows_fwd(const Params& p, int dtype, cudaStream_t st);
constexpr int kTcPad = 384;  // (lse, delta) rows are padded to a multiple of every tile height

}  // namespace bias_attn
}  // namespace b2
