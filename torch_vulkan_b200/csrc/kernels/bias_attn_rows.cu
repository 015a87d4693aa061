// Relative-position-bias attention for a few query rows (a decoder's new tokens against its cache): forward on the FMA
// pipe, bound by reading K and V once.
//
// A block owns one key/value head and a range of keys, for all query rows that read them (Sq x the heads that share the
// head, at most 8). A key's row of K is spread over LPK lanes, 16 bytes each, so a warp takes 32 / LPK keys at a time and
// U such groups of K and V are loaded before the first is used. Every group of lanes keeps its own running maximum, sum
// and output in fp32; they are joined through shared memory at the end, and the blocks of a head by the combine kernel.
// A tensor-core tile would spend 128 rows of exponentials on these few: 74 us against 54 for one row of 8 x 16 heads over 8192
// keys of 64 (268 MB of K and V, 41 us at the measured memory rate).
#include "bias_attn.cuh"
#include "tc_ptx.cuh"

namespace b2 {
namespace bias_attn {
namespace {

constexpr int NW = 4;  // warps per block

template <typename T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);
  static __device__ __forceinline__ void unpack(const uint4& raw, float* f) {
    const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32<T>(t[i]);
  }
};

// R: query rows (Sq * G rounded up to a power of two); LPK: lanes per key.
template <typename T, int R, int LPK>
__global__ void __launch_bounds__(NW * 32) rows_kernel(const __grid_constant__ Params p, int rows) {
  constexpr int N = Vec16<T>::N, KPW = 32 / LPK, U = R >= 4 ? 2 : 4;
  extern __shared__ float sm[];
  float* bias = sm;  // [G][2R + 1] of the block's heads, later the joined outputs
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane / LPK, part = lane % LPK;
  const int b = (int)blockIdx.x / p.Hk, hk = (int)blockIdx.x % p.Hk, G = p.H / p.Hk;
  tc::pdl_wait();
  tc::pdl_trigger();
  const int vl = 2 * p.R + 1;
  const int end = key_end(p, p.Sq - 1);
  const int per = ((end + p.nsplit - 1) / p.nsplit + NW * KPW * U - 1) / (NW * KPW * U) * (NW * KPW * U);
  const int j0 = (int)min((int64_t)end, (int64_t)blockIdx.y * per), j1 = min(end, j0 + per);
  // the part of the bias that these keys reach: a single entry for keys wholly beyond max_distance
  const int lo = max(-p.R, min(p.R, j0 - (p.Sq - 1) - p.q_off)), span = max(-p.R, min(p.R, j1 - 1 - p.q_off)) - lo + 1;
  for (int i = threadIdx.x; i < G * span; i += NW * 32) {
    const int g = i / span, rel = lo + i - g * span;
    bias[g * vl + rel + p.R] = bias_at(p, hk * G + g, rel);
  }

  // this lane's slice of the queries, scaled into log2 units; row r is query r % Sq of head hk * G + r / Sq
  const bool has = part * N < p.D;
  float q[R][N];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r < rows && has) {
      const uint4 raw = *reinterpret_cast<const uint4*>(row_of<T>(p.q, p.q_s, b, hk * G + r / p.Sq, r % p.Sq) + part * N);
      Vec16<T>::unpack(raw, q[r]);
#pragma unroll
      for (int i = 0; i < N; ++i) q[r][i] *= p.scale * kLog2e;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) q[r][i] = 0.f;
    }
  }
  __syncthreads();

  float m[R], l[R], acc[R][N];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[r][i] = 0.f;
  }
  const T* kb = row_of<T>(p.k, p.k_s, b, hk, 0) + part * N;
  const T* vb = row_of<T>(p.v, p.v_s, b, hk, 0) + part * N;
  for (int j = j0 + warp * KPW * U; j < j1; j += NW * KPW * U) {  // the same trip count for the whole warp
    uint4 kr[U], vr[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j + u * KPW + sub;
      on[u] = key < j1 && (p.mask == nullptr || p.mask[(int64_t)b * p.mask_sb + key] != 0);
      const bool ld = on[u] && has;  // what a masked key holds is not read
      kr[u] = ld ? __ldcs(reinterpret_cast<const uint4*>(kb + (int64_t)key * p.k_s[2])) : make_uint4(0u, 0u, 0u, 0u);
      vr[u] = ld ? __ldcs(reinterpret_cast<const uint4*>(vb + (int64_t)key * p.v_s[2])) : make_uint4(0u, 0u, 0u, 0u);
    }
    float s[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float kf[N];
      Vec16<T>::unpack(kr[u], kf);
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float d = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) d = fmaf(q[r][i], kf[i], d);
#pragma unroll
        for (int o = LPK / 2; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
        const int rel = j + u * KPW + sub - (r % p.Sq) - p.q_off;
        const bool ok = on[u] && r < rows && !(p.causal && rel > 0);
        s[u][r] = ok ? d + bias[(r / p.Sq) * vl + max(-p.R, min(p.R, rel)) + p.R] : -INFINITY;
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float mx = m[r];
#pragma unroll
      for (int u = 0; u < U; ++u) mx = fmaxf(mx, s[u][r]);
      const float ref = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: exp2(-inf - 0) = 0
      const float alpha = exp2f(m[r] - ref);
      m[r] = mx;
      l[r] *= alpha;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[r][i] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) s[u][r] = exp2f(s[u][r] - ref), l[r] += s[u][r];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float vf[N];
      Vec16<T>::unpack(vr[u], vf);
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[r][i] = fmaf(s[u][r], vf[i], acc[r][i]);
    }
  }
  // ---- join the NW * KPW groups of lanes of every row ----
  __syncthreads();  // the bias is done with
  constexpr int GRP = NW * KPW;
  float* so = sm;                         // [GRP][LPK * N]
  float* sml = so + GRP * LPK * N;        // [GRP][2]
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (r >= rows) break;
    const int grp = warp * KPW + sub;
#pragma unroll
    for (int i = 0; i < N; ++i) so[grp * (LPK * N) + part * N + i] = acc[r][i];
    if (part == 0) sml[2 * grp] = m[r], sml[2 * grp + 1] = l[r];
    __syncthreads();
    float M = -INFINITY;
#pragma unroll
    for (int g = 0; g < GRP; ++g) M = fmaxf(M, sml[2 * g]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f;
#pragma unroll
    for (int g = 0; g < GRP; ++g) L = fmaf(sml[2 * g + 1], exp2f(sml[2 * g] - ref), L);
    const int h = hk * G + r / p.Sq, i = r % p.Sq;
    const int64_t row = ((int64_t)b * p.H + h) * p.Sq + i;
    const int64_t prow = (int64_t)blockIdx.y * p.B * p.H * p.Sq + row;
    for (int d = threadIdx.x; d < p.D; d += NW * 32) {
      float o = 0.f;
#pragma unroll
      for (int g = 0; g < GRP; ++g) o = fmaf(so[g * (LPK * N) + d], exp2f(sml[2 * g] - ref), o);
      if (p.nsplit > 1) {
        p.part_o[prow * p.D + d] = o;
      } else {
        o = L > 0.f ? o / L : 0.f;
        row_of<T>(p.o, p.o_s, b, h, i)[d] = from_f32<T>(o);
        if (p.o32) p.o32[row * p.D + d] = o;
      }
    }
    if (threadIdx.x == 0) {
      if (p.nsplit > 1) p.part_ml[prow] = make_float2(M, L);
      else if (p.lse) p.lse[row] = L > 0.f ? (M + log2f(L)) * kLn2 : -INFINITY;
    }
    __syncthreads();
  }
}

template <typename T, int R, int LPK>
int launch(const Params& p, int rows, cudaStream_t st) {
  constexpr int N = Vec16<T>::N, GRP = NW * 32 / LPK;
  const int G = p.H / p.Hk;
  const int smem = std::max(G * (2 * p.R + 1), GRP * (LPK * N + 2)) * 4;
  if (int rc = allow_smem<rows_kernel<T, R, LPK>>(smem, "bias_attn_rows")) return rc;
  return launch_pdl("bias_attn_rows", rows_kernel<T, R, LPK>, dim3(p.B * p.Hk, p.nsplit), dim3(NW * 32), smem, st, p, rows);
}

template <typename T, int R>
int by_width(const Params& p, int rows, cudaStream_t st) {
  const int lanes = (p.D + Vec16<T>::N - 1) / Vec16<T>::N;
  if (lanes <= 4) return launch<T, R, 4>(p, rows, st);
  if (lanes <= 8) return launch<T, R, 8>(p, rows, st);
  if (lanes <= 16) return launch<T, R, 16>(p, rows, st);
  return launch<T, R, 32>(p, rows, st);
}
template <typename T>
int by_rows(const Params& p, cudaStream_t st) {
  const int rows = p.Sq * (p.H / p.Hk);
  if (rows <= 1) return by_width<T, 1>(p, rows, st);
  if (rows <= 2) return by_width<T, 2>(p, rows, st);
  if (rows <= 4) return by_width<T, 4>(p, rows, st);
  return by_width<T, 8>(p, rows, st);
}

}  // namespace

// At most 8 query rows per key/value head, and rows that are whole aligned 16-byte groups.
bool rows_eligible(const b2_bias_attn_args* a) {
  const int64_t es = (int64_t)dtype_size(a->dtype), n = 16 / es;
  auto ok = [&](const void* t, const int64_t* s) {
    return ((uintptr_t)t & 15) == 0 && s[0] % n == 0 && s[1] % n == 0 && s[2] % n == 0;
  };
  return a->Sk >= 1 && a->Sq * (a->H / a->Hk) <= 8 && a->D % n == 0 && ok(a->q, a->q_s) && ok(a->k, a->k_s) && ok(a->v, a->v_s);
}

int rows_fwd(const Params& p, int dtype, cudaStream_t st) {
  switch (dtype) {
    case B2_F32: return by_rows<float>(p, st);
    case B2_BF16: return by_rows<__nv_bfloat16>(p, st);
    default: return by_rows<__half>(p, st);
  }
}

}  // namespace bias_attn
}  // namespace b2
