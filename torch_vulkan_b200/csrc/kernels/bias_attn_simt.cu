// Relative-position-bias attention on the FMA pipe: fp32 inputs, and 16-bit inputs whose layout the tensor-core
// kernels do not take. A block of 128 threads owns 32 rows and walks the other side in tiles of 64, held in shared memory
// as fp32, each thread on 4 x 4 scores and on 4 rows x DP / 16 columns of the outputs; every operand read is a 16-byte shared-memory load
// whose bank pattern is conflict-free (rows padded by 4 floats). Forward: one pass with the running maximum and sum,
// the key axis split over blockIdx.z when there are few query tiles. Backward: one kernel owns query tiles (dQ and the
// bias gradient), one owns key tiles (dK, dV, summed over the query heads that share them), so every sum has one owner
// and a fixed order.
#include "bias_attn.cuh"

namespace b2 {
namespace bias_attn {
namespace {

constexpr int OWN = kSimtTile, T64 = 64;  // rows a block owns, rows of a walked tile
constexpr int NTH = OWN / 4 * 16;         // threads
constexpr int PS = T64 + 4;

template <int DP>
struct Smem {
  static constexpr int LD = DP + 4;
  static constexpr int TILE = T64 * LD, OTILE = OWN * LD;  // floats of a walked and of an owned operand tile
};

// ROWS rows of an operand -> fp32 tile, zeros past the end of the rows, past D, and (keep != NULL) in masked rows. Rows of
// whole aligned 16-byte groups are read so.
template <typename T, int DP, int ROWS>
__device__ __forceinline__ void load_tile(float* dst, const void* base, const int64_t* s, int b, int h, int r0, int rows,
                                          int D, float mul, const uint8_t* keep) {
  constexpr int V = 16 / (int)sizeof(T);
  const T* origin = row_of<T>(base, s, b, h, r0);
  if (D % V == 0 && s[2] % V == 0 && ((uintptr_t)origin & 15) == 0) {
#pragma unroll 4
    for (int e = threadIdx.x; e < ROWS * (DP / V); e += NTH) {
      const int r = e / (DP / V), d = e % (DP / V) * V;
      uint4 raw = make_uint4(0u, 0u, 0u, 0u);
      if (r0 + r < rows && d < D && (keep == nullptr || keep[r])) raw = *reinterpret_cast<const uint4*>(origin + r * s[2] + d);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < V; ++i) dst[r * Smem<DP>::LD + d + i] = to_f32<T>(t[i]) * mul;
    }
    return;
  }
  for (int e = threadIdx.x; e < ROWS * DP; e += NTH) {
    const int r = e / DP, d = e % DP;
    float v = 0.f;
    if (r0 + r < rows && d < D && (keep == nullptr || keep[r])) v = to_f32<T>(origin[r * s[2] + d]) * mul;
    dst[r * Smem<DP>::LD + d] = v;
  }
}

// acc[i][j] += A[ty*4 + i] . B[tx + 16 j] over DP columns
template <int DP>
__device__ __forceinline__ void dot_tile(const float* A, const float* B, int ty, int tx, float (&acc)[4][4]) {
  constexpr int LD = Smem<DP>::LD;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 a[4], c[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4*>(A + (ty * 4 + i) * LD + d);
#pragma unroll
    for (int j = 0; j < 4; ++j) c[j] = *reinterpret_cast<const float4*>(B + (tx + 16 * j) * LD + d);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        acc[i][j] = fmaf(a[i].x, c[j].x, acc[i][j]);
        acc[i][j] = fmaf(a[i].y, c[j].y, acc[i][j]);
        acc[i][j] = fmaf(a[i].z, c[j].z, acc[i][j]);
        acc[i][j] = fmaf(a[i].w, c[j].w, acc[i][j]);
      }
  }
}

// acc[i][c*4 + e] += sum_k P[ty*4 + i][k] * V[k][tx*4 + 64 c + e]
template <int DP>
__device__ __forceinline__ void pv_tile(const float* P, const float* V, int ty, int tx, float (&acc)[4][DP / 16]) {
  constexpr int LD = Smem<DP>::LD;
#pragma unroll 2
  for (int k = 0; k < T64; k += 4) {
    float4 pr[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) pr[i] = *reinterpret_cast<const float4*>(P + (ty * 4 + i) * PS + k);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int c = 0; c < DP / 64; ++c) {
        const float4 w = *reinterpret_cast<const float4*>(V + (k + kk) * LD + tx * 4 + 64 * c);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float pv = reinterpret_cast<const float*>(&pr[i])[kk];
          acc[i][c * 4 + 0] = fmaf(pv, w.x, acc[i][c * 4 + 0]);
          acc[i][c * 4 + 1] = fmaf(pv, w.y, acc[i][c * 4 + 1]);
          acc[i][c * 4 + 2] = fmaf(pv, w.z, acc[i][c * 4 + 2]);
          acc[i][c * 4 + 3] = fmaf(pv, w.w, acc[i][c * 4 + 3]);
        }
      }
  }
}

__device__ __forceinline__ float max16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float sum16(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// keep[j] for the n keys from k0, of which those from `end` on are hidden from every query that is asked about; returns
// whether any is left.
__device__ __forceinline__ bool load_keep(const Params& p, int b, int k0, int n, int end, uint8_t* keep) {
  bool any = false;
  if ((int)threadIdx.x < n) {
    const int j = k0 + threadIdx.x;
    const bool ok = j < end && (p.mask == nullptr || p.mask[(int64_t)b * p.mask_sb + j] != 0);
    keep[threadIdx.x] = ok;
    any = ok;
  }
  return __syncthreads_or(any);
}

__device__ __forceinline__ void fill_bias(const Params& p, int h, float* bias) {
  for (int i = threadIdx.x; i <= 2 * p.R; i += NTH) bias[i] = bias_at(p, h, i - p.R);
}
__device__ __forceinline__ float bias_get(const Params& p, const float* bias, int rel) {
  if (p.causal && rel > 0) return -INFINITY;
  return bias[max(-p.R, min(p.R, rel)) + p.R];
}

template <typename T, int DP>
__global__ void __launch_bounds__(NTH) fwd_kernel(const __grid_constant__ Params p) {
  extern __shared__ float4 sm4[];
  float* Qs = reinterpret_cast<float*>(sm4);
  float* Ks = Qs + Smem<DP>::OTILE;
  float* Vs = Ks + Smem<DP>::TILE;
  float* Ps = Vs + Smem<DP>::TILE;
  float* bias = Ps + OWN * PS;
  uint8_t* keep = reinterpret_cast<uint8_t*>(bias + 2 * p.R + 1);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int q0 = blockIdx.x * OWN;
  const int b = blockIdx.y / p.H, h = blockIdx.y % p.H, hk = h / (p.H / p.Hk);
  fill_bias(p, h, bias);
  load_tile<T, DP, OWN>(Qs, p.q, p.q_s, b, h, q0, p.Sq, p.D, p.scale * kLog2e, nullptr);
  float m[4], l[4], acc[4][DP / 16];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[i][c] = 0.f;
  }
  const int end = key_end(p, min(q0 + OWN, p.Sq) - 1), nt = (end + T64 - 1) / T64;
  const int per = (nt + p.nsplit - 1) / p.nsplit;
  const int t1 = min(nt, ((int)blockIdx.z + 1) * per);
  for (int t = blockIdx.z * per; t < t1; ++t) {
    const int k0 = t * T64;
    __syncthreads();
    if (!load_keep(p, b, k0, T64, end, keep)) continue;
    load_tile<T, DP, T64>(Ks, p.k, p.k_s, b, hk, k0, p.Sk, p.D, 1.f, keep);
    load_tile<T, DP, T64>(Vs, p.v, p.v_s, b, hk, k0, p.Sk, p.D, 1.f, keep);
    __syncthreads();
    float s[4][4] = {};
    dot_tile<DP>(Qs, Ks, ty, tx, s);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int qi = q0 + ty * 4 + i;
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = tx + 16 * j;
        s[i][j] = keep[c] ? s[i][j] + bias_get(p, bias, k0 + c - qi - p.q_off) : -INFINITY;
        mx = fmaxf(mx, s[i][j]);
      }
      mx = fmaxf(m[i], max16(mx));
      const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: exp2(-inf - 0) = 0
      const float alpha = exp2f(m[i] - ref);
      m[i] = mx;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float e = exp2f(s[i][j] - ref);
        Ps[(ty * 4 + i) * PS + tx + 16 * j] = e;
        sum += e;
      }
      l[i] = l[i] * alpha + sum16(sum);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) acc[i][c] *= alpha;
    }
    __syncwarp();  // a warp's 8 rows of P are read by the same warp
    pv_tile<DP>(Ps, Vs, ty, tx, acc);
  }
  const int64_t nrow = (int64_t)p.B * p.H * p.Sq;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = q0 + ty * 4 + i;
    if (qi >= p.Sq) continue;
    const int64_t row = (int64_t)blockIdx.y * p.Sq + qi;
    if (p.nsplit > 1) {
      const int64_t pr = (int64_t)blockIdx.z * nrow + row;
      if (tx == 0) p.part_ml[pr] = make_float2(m[i], l[i]);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const int d = tx * 4 + 64 * (c >> 2) + (c & 3);
        if (d < p.D) p.part_o[pr * p.D + d] = acc[i][c];
      }
    } else {
      const float inv = inverse_sum(l[i]);
      T* o = row_of<T>(p.o, p.o_s, b, h, qi);
#pragma unroll
      for (int c = 0; c < DP / 16; ++c) {
        const int d = tx * 4 + 64 * (c >> 2) + (c & 3);
        if (d < p.D) {
          o[d] = from_f32<T>(acc[i][c] * inv);
          if (p.o32) p.o32[row * p.D + d] = acc[i][c] * inv;
        }
      }
      if (tx == 0 && p.lse) p.lse[row] = log_sum(m[i], l[i]);
    }
  }
}

// dQ and the bias gradient: a block owns 32 query rows of one head and walks the keys.
template <typename T, int DP>
__device__ __forceinline__ void dq_side(const Params& p, int block, int xtiles) {
  extern __shared__ float4 sm4[];
  float* Qs = reinterpret_cast<float*>(sm4);
  float* Gs = Qs + Smem<DP>::OTILE;  // dO
  float* Ks = Gs + Smem<DP>::OTILE;
  float* Vs = Ks + Smem<DP>::TILE;
  float* Ps = Vs + Smem<DP>::TILE;  // dS
  float* bias = Ps + OWN * PS;
  float* diag = bias + 2 * p.R + 1;                       // 95 diagonal sums of a tile
  int* dbk = reinterpret_cast<int*>(diag + 2 * T64);      // and their buckets
  uint8_t* keep = reinterpret_cast<uint8_t*>(dbk + 2 * T64);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int bh = block / xtiles, q0 = (block - bh * xtiles) * OWN;
  const int b = bh / p.H, h = bh % p.H, hk = h / (p.H / p.Hk);
  fill_bias(p, h, bias);
  load_tile<T, DP, OWN>(Qs, p.q, p.q_s, b, h, q0, p.Sq, p.D, p.scale * kLog2e, nullptr);
  load_tile<T, DP, OWN>(Gs, p.d_o, p.do_s, b, h, q0, p.Sq, p.D, 1.f, nullptr);
  float L[4], dl[4], acc[4][DP / 16];
  const int end = key_end(p, min(q0 + OWN, p.Sq) - 1), nt = (end + T64 - 1) / T64;
  const Visible seen = visible_keys(p, b, end, 0, 0, NTH, reinterpret_cast<int*>(diag));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = q0 + ty * 4 + i;
    const int64_t row = (int64_t)bh * p.Sq + qi;
    // rows past the end and rows with no key: exp2(x - inf) = 0
    L[i] = qi < p.Sq ? p.lse[row] * kLog2e : INFINITY;
    if (L[i] == -INFINITY) L[i] = INFINITY;
    dl[i] = qi < p.Sq ? p.delta[row] : 0.f;
    if (sees_one(p, qi, seen.first, seen.second) && isfinite(L[i] + dl[i])) L[i] = INFINITY;  // dS = 0; a NaN goes its way
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) acc[i][c] = 0.f;
  }
  float db = 0.f;  // thread n: sum of dS over bucket n
  for (int t = 0; t < nt; ++t) {
    const int k0 = t * T64;
    __syncthreads();
    if (!load_keep(p, b, k0, T64, end, keep)) continue;
    load_tile<T, DP, T64>(Ks, p.k, p.k_s, b, hk, k0, p.Sk, p.D, 1.f, keep);
    load_tile<T, DP, T64>(Vs, p.v, p.v_s, b, hk, k0, p.Sk, p.D, 1.f, keep);
    __syncthreads();
    float s[4][4] = {}, dp[4][4] = {};
    dot_tile<DP>(Qs, Ks, ty, tx, s);
    dot_tile<DP>(Gs, Vs, ty, tx, dp);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int qi = q0 + ty * 4 + i;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = tx + 16 * j;
        const float x = keep[c] ? s[i][j] + bias_get(p, bias, k0 + c - qi - p.q_off) : -INFINITY;
        Ps[(ty * 4 + i) * PS + c] = exp2f(x - L[i]) * (dp[i][j] - dl[i]);
      }
    }
    if (p.dtab) {
      __syncthreads();
      if (threadIdx.x < OWN + T64 - 1) {
        const int d = (int)threadIdx.x - (OWN - 1);  // key - query inside the tile
        float a = 0.f;
        for (int r = max(0, -d); r < min(OWN, T64 - d); ++r) a += Ps[r * PS + r + d];
        diag[threadIdx.x] = a;
        dbk[threadIdx.x] = bucket_of(p, max(-p.R, min(p.R, k0 + d - q0 - p.q_off)));
      }
      __syncthreads();
      if ((int)threadIdx.x < p.nb)
        for (int i = 0; i < OWN + T64 - 1; ++i) db += dbk[i] == (int)threadIdx.x ? diag[i] : 0.f;
    } else {
      __syncwarp();
    }
    pv_tile<DP>(Ps, Ks, ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int qi = q0 + ty * 4 + i;
    if (qi >= p.Sq || !p.dq) continue;
    T* o = row_of<T>(p.dq, p.dq_s, b, h, qi);
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = tx * 4 + 64 * (c >> 2) + (c & 3);
      if (d < p.D) o[d] = from_f32<T>(acc[i][c] * p.scale);
    }
  }
  if (p.dtab && (int)threadIdx.x < p.nb)
    p.dtab[(int64_t)block * p.nb + threadIdx.x] = db;
}

// dK, dV: a block owns 32 keys of one key/value head and walks the queries of every head that shares it.
template <typename T, int DP>
__device__ __forceinline__ void dkv_side(const Params& p, int block, int xtiles) {
  extern __shared__ float4 sm4[];
  float* Ks = reinterpret_cast<float*>(sm4);
  float* Vs = Ks + Smem<DP>::OTILE;
  float* Qs = Vs + Smem<DP>::OTILE;
  float* Gs = Qs + Smem<DP>::TILE;  // dO
  float* Pt = Gs + Smem<DP>::TILE;  // P^T
  float* St = Pt + OWN * PS;        // dS^T
  float* bias = St + OWN * PS;
  float* Lq = bias + 2 * p.R + 1;
  float* Dq = Lq + T64;
  uint8_t* keep = reinterpret_cast<uint8_t*>(Dq + T64);
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int bh = block / xtiles, k0 = (block - bh * xtiles) * OWN;
  const int b = bh / p.Hk, hk = bh % p.Hk, G = p.H / p.Hk;
  const bool some = load_keep(p, b, k0, OWN, key_end(p, p.Sq - 1), keep);
  load_tile<T, DP, OWN>(Ks, p.k, p.k_s, b, hk, k0, p.Sk, p.D, 1.f, keep);
  load_tile<T, DP, OWN>(Vs, p.v, p.v_s, b, hk, k0, p.Sk, p.D, 1.f, keep);
  float dk[4][DP / 16] = {}, dv[4][DP / 16] = {};
  // causal: the first query row that sees key k0
  const int64_t first = p.causal ? max((int64_t)0, (int64_t)k0 - p.q_off) : 0;
  const int nt = (p.Sq + T64 - 1) / T64;
  for (int g = 0; g < G && some; ++g) {
    const int h = hk * G + g;
    __syncthreads();
    fill_bias(p, h, bias);
    for (int t = (int)min((int64_t)nt, first / T64); t < nt; ++t) {
      const int q0 = t * T64;
      __syncthreads();
      load_tile<T, DP, T64>(Qs, p.q, p.q_s, b, h, q0, p.Sq, p.D, 1.f, nullptr);
      load_tile<T, DP, T64>(Gs, p.d_o, p.do_s, b, h, q0, p.Sq, p.D, 1.f, nullptr);
      if (threadIdx.x < T64) {
        const int qi = q0 + threadIdx.x;
        const int64_t row = ((int64_t)b * p.H + h) * p.Sq + qi;
        float L = qi < p.Sq ? p.lse[row] * kLog2e : INFINITY;
        Lq[threadIdx.x] = L == -INFINITY ? INFINITY : L;
        Dq[threadIdx.x] = qi < p.Sq ? p.delta[row] : 0.f;
      }
      __syncthreads();
      float s[4][4] = {}, dp[4][4] = {};
      dot_tile<DP>(Ks, Qs, ty, tx, s);
      dot_tile<DP>(Vs, Gs, ty, tx, dp);
      const float sl2 = p.scale * kLog2e;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = ty * 4 + i;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = tx + 16 * j;
          const float x = keep[r] ? fmaf(s[i][j], sl2, bias_get(p, bias, k0 + r - (q0 + c) - p.q_off)) : -INFINITY;
          const float e = exp2f(x - Lq[c]);
          Pt[r * PS + c] = e;
          St[r * PS + c] = e * (dp[i][j] - Dq[c]);
        }
      }
      __syncwarp();
      pv_tile<DP>(Pt, Gs, ty, tx, dv);
      pv_tile<DP>(St, Qs, ty, tx, dk);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int kj = k0 + ty * 4 + i;
    if (kj >= p.Sk) continue;
#pragma unroll
    for (int c = 0; c < DP / 16; ++c) {
      const int d = tx * 4 + 64 * (c >> 2) + (c & 3);
      if (d >= p.D) continue;
      if (p.dk) row_of<T>(p.dk, p.dk_s, b, hk, kj)[d] = from_f32<T>(dk[i][c] * p.scale);
      if (p.dv) row_of<T>(p.dv, p.dv_s, b, hk, kj)[d] = from_f32<T>(dv[i][c]);
    }
  }
}

// Both sides in one launch, the key blocks (the longer walks) first: either alone leaves SMs idle at these sizes.
template <typename T, int DP>
__global__ void __launch_bounds__(NTH) bwd_kernel(const __grid_constant__ Params p, int key_blocks, int key_tiles, int query_tiles) {
  if ((int)blockIdx.x < key_blocks) dkv_side<T, DP>(p, blockIdx.x, key_tiles);
  else dq_side<T, DP>(p, (int)blockIdx.x - key_blocks, query_tiles);
}

template <int DP>
int smem_bytes(const Params& p, int own, int walked, int ps) {
  return (own * Smem<DP>::OTILE + walked * Smem<DP>::TILE + ps * OWN * PS + 2 * p.R + 1 + 4 * T64 + 4) * 4 + T64;
}

// Plain launches: these blocks are far fewer than the SMs could hold, and blocks that start early, beside a kernel that is
// still draining, are packed onto the SMs that are free (157 us a step instead of 113 at 203 x 331 x 40, 6 heads).
template <typename T, int DP>
int fwd_t(const Params& p, cudaStream_t st) {
  const int sm = smem_bytes<DP>(p, 1, 2, 1);
  if (int rc = allow_smem<fwd_kernel<T, DP>>(sm, "bias_attn_fwd_simt")) return rc;
  {
    LaunchScope ls("bias_attn_fwd_simt", st);
    dim3 grid((p.Sq + OWN - 1) / OWN, p.B * p.H, p.nsplit);
    fwd_kernel<T, DP><<<grid, NTH, sm, st>>>(p);
  }
  return after_launch("bias_attn_fwd_simt");
}

template <typename T, int DP>
int bwd_t(const Params& p, cudaStream_t st) {
  const int ktiles = (p.Sk + OWN - 1) / OWN, qtiles = (p.Sq + OWN - 1) / OWN;
  const int64_t kblocks = p.dk || p.dv ? (int64_t)p.B * p.Hk * ktiles : 0;
  const int64_t qblocks = p.dq || p.dtab ? (int64_t)p.B * p.H * qtiles : 0;
  if (kblocks + qblocks == 0) return 0;
  if (kblocks + qblocks >= (1ll << 31)) return fail(B2_ERR_ARG, "bias_attn_bwd: too many tiles");
  const int sm = kblocks ? smem_bytes<DP>(p, 2, 2, 2) : smem_bytes<DP>(p, 2, 2, 1);
  if (int rc = allow_smem<bwd_kernel<T, DP>>(sm, "bias_attn_bwd_simt")) return rc;
  {
    LaunchScope ls("bias_attn_bwd_simt", st);
    bwd_kernel<T, DP><<<(unsigned)(kblocks + qblocks), NTH, sm, st>>>(p, (int)kblocks, ktiles, qtiles);
  }
  return after_launch("bias_attn_bwd_simt");
}

template <typename T>
int fwd_d(const Params& p, cudaStream_t st) {
  return p.D <= 64 ? fwd_t<T, 64>(p, st) : fwd_t<T, 128>(p, st);
}
template <typename T>
int bwd_d(const Params& p, cudaStream_t st) {
  return p.D <= 64 ? bwd_t<T, 64>(p, st) : bwd_t<T, 128>(p, st);
}

}  // namespace

int simt_fwd(const Params& p, int dtype, cudaStream_t st) {
  switch (dtype) {
    case B2_F32: return fwd_d<float>(p, st);
    case B2_BF16: return fwd_d<__nv_bfloat16>(p, st);
    default: return fwd_d<__half>(p, st);
  }
}
int simt_bwd(const Params& p, int dtype, cudaStream_t st) {
  switch (dtype) {
    case B2_F32: return bwd_d<float>(p, st);
    case B2_BF16: return bwd_d<__nv_bfloat16>(p, st);
    default: return bwd_d<__half>(p, st);
  }
}

}  // namespace bias_attn
}  // namespace b2
