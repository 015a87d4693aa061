// Relative-position-bias attention for a few query rows (a decoder's new tokens against its cache): forward, bound by
// reading K and V once.
//
// A block owns one key/value head, a range of keys, and up to 8 of the query rows that read them (Sq x the heads that share
// the head). Blocks of the same keys are neighbours, so that the keys come from memory once and from L2 after that. The
// ranges of a row are joined by the combine kernel.
//
// 16-bit types: rows_mma_kernel. The keys are the 16 rows of an m16n8k16 product and the query rows its 8 columns,
// S^T = K Q^T and O^T = V^T P^T, so that 8 query rows cost what one does and nothing is computed for rows that are not
// there. (A tcgen05 tile has 128 rows of keys or of queries: with the queries as its rows it spends 128 rows of
// exponentials on these few, 79 us for the case below.) Each warp copies its own tiles of 16 keys through a ring in shared
// memory, without a barrier of the block, and keeps its own reference, sum and O^T in fp32 until the end. P enters the second
// product as its rounded value plus the rounded rest, so that P is good to 2^-17 and the sums are fp32.
// One row of 8 x 16 heads over 8192 keys of 64 (268 MB of K and V, 41 us at the measured memory rate): 48 us with the join;
// products on the FMA pipe, 16 bytes of a key per lane, took 57 us, and for 8 rows of 4 x 4 key/value heads over 16384 keys
// of 128 (134 MB) 260 us against 31. A ring of two tiles leaves six blocks to an SM: 50 us against 56 with three tiles and
// 58 with four.
//
// fp32: rows_kernel, on the FMA pipe. A key's row of K is spread over LPK lanes, 16 bytes each, so a warp takes 32 / LPK
// keys at a time and U such groups of K and V are loaded before the first is used. Every group of lanes keeps its own running
// maximum, sum and output; they are joined through shared memory at the end.
#include "bias_attn.cuh"
#include "tc_ptx.cuh"

namespace b2 {
namespace bias_attn {
namespace {

constexpr int NW = 4;  // warps per block

constexpr int ST = 2;      // tiles of a warp's ring, one of them in use
constexpr int KT = 16;     // keys per tile
static_assert(ST * KT == 32, "the seen keys of a ring are kept as the bits of one word");
constexpr float kLift = 7.f, kSlack = 8.f;  // of the exponentials' reference, see below

// 16 bytes from memory into shared memory, or zeros without a read.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void load_frag(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void load_frag_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  T t[2] = {from_f32<T>(a), from_f32<T>(b)};
  return *reinterpret_cast<uint32_t*>(t);
}
// (a, b) rounded, and what the rounding left, rounded.
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(a, b);
  const T* t = reinterpret_cast<const T*>(&hi);
  lo = pack2<T>(a - to_f32<T>(t[0]), b - to_f32<T>(t[1]));
}

// KD: 16-wide steps of the head dimension.
template <typename T, int KD>
__global__ void __launch_bounds__(NW * 32) rows_mma_kernel(const __grid_constant__ Params p, int groups) {
  constexpr int CH = 2 * KD, RB = CH * 16, DP = KD * 16, TILE = KT * RB, PASS = 32 / CH, STEP = NW * KT;
  extern __shared__ __align__(128) uint8_t smem[];
  float* bias = reinterpret_cast<float*>(smem + NW * ST * 2 * TILE);  // [heads][2R + 1] of the heads of the block's rows
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int bh = (int)blockIdx.x / groups, b = bh / p.Hk, hk = bh % p.Hk, G = p.H / p.Hk;
  const int first = (int)blockIdx.x % groups * 8, rows = min(8, p.Sq * G - first);
  const int h0 = first / p.Sq, nh = (first + rows - 1) / p.Sq - h0 + 1;  // the heads of these rows, after hk * G
  tc::pdl_wait();
  tc::pdl_trigger();
  const int vl = 2 * p.R + 1;
  const int end = key_end(p, p.Sq - 1);
  const int per = ((end + p.nsplit - 1) / p.nsplit + STEP - 1) / STEP * STEP;
  const int j0 = (int)min((int64_t)end, (int64_t)blockIdx.y * per), j1 = min(end, j0 + per);

  // ---- a warp's own ring of K and V tiles; 16-byte chunk c of row r lies at chunk c ^ (r & 7) ----
  const uint32_t ring = tc::smem_u32(smem) + warp * (ST * 2 * TILE);
  const int crow = lane / CH, cch = lane % CH;
  const bool has = cch * 8 < p.D;
  const T* kb = row_of<T>(p.k, p.k_s, b, hk, 0) + cch * 8;
  const T* vb = row_of<T>(p.v, p.v_s, b, hk, 0) + cch * 8;
  const uint8_t* mb = p.mask ? p.mask + (int64_t)b * p.mask_sb : nullptr;
  auto see = [&](int j) {  // whether key j + lane % 16 is read
    const int key = j + (lane & 15);
    return key < j1 && (mb == nullptr || mb[key] != 0);
  };
  uint32_t live = 0;  // 16 bits for each tile in the ring, the oldest lowest
  bool seen = see(j0 + warp * KT);
  auto fetch = [&](int j, int slot) {
    const uint32_t bits = __ballot_sync(0xffffffffu, seen) & 0xffffu;
    seen = see(j + STEP);  // the next tile's, so that its latency is hidden
    if (bits) {
#pragma unroll
      for (int i = 0; i < KT / PASS; ++i) {
        const int r = i * PASS + crow;
        const bool on = has && (bits >> r & 1u);  // what a masked key holds is not read
        const int at = on ? j + r : j;
        const uint32_t dst = ring + slot * (2 * TILE) + r * RB + ((cch ^ (r & 7)) << 4);
        copy16(dst, on ? kb + (int64_t)at * p.k_s[2] : kb, on);
        copy16(dst + TILE, on ? vb + (int64_t)at * p.v_s[2] : vb, on);
      }
    }
    copy_commit();
    live = live >> 16 | bits << 16;
  };
  const int jw = j0 + warp * KT;
#pragma unroll
  for (int n = 0; n < ST - 1; ++n) fetch(jw + n * STEP, n);

  // the part of the bias that these keys reach: a single entry for keys wholly beyond max_distance
  const int lo = max(-p.R, min(p.R, j0 - (p.Sq - 1) - p.q_off)), span = max(-p.R, min(p.R, j1 - 1 - p.q_off)) - lo + 1;
  for (int i = threadIdx.x; i < nh * span; i += NW * 32) {
    const int h = i / span, rel = lo + i - h * span;
    bias[h * vl + rel + p.R] = bias_at(p, hk * G + h0 + h, rel);
  }
  // Q^T as the second operand: this lane holds dims 16 k + 2 t (+ 1, + 8, + 9) of row g; row r is query (first + r) % Sq
  // of head hk * G + (first + r) / Sq
  uint32_t q[KD][2];
  {
    const int r = first + min(g, rows - 1);
    const T* qr = row_of<T>(p.q, p.q_s, b, hk * G + r / p.Sq, r % p.Sq);
#pragma unroll
    for (int k = 0; k < KD; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = 16 * k + 8 * i + 2 * t;
        q[k][i] = g < rows && d < p.D ? *reinterpret_cast<const uint32_t*>(qr + d) : 0u;
      }
  }
  const int r0 = 2 * t, r1 = 2 * t + 1;  // the two rows whose scores this lane holds
  const bool ok0 = r0 < rows, ok1 = r1 < rows;
  const float* b0 = bias + min((first + r0) / p.Sq - h0, nh - 1) * vl + p.R;
  const float* b1 = bias + min((first + r1) / p.Sq - h0, nh - 1) * vl + p.R;
  const int e0 = (first + r0) % p.Sq + p.q_off, e1 = (first + r1) % p.Sq + p.q_off;
  const float sc = p.scale * kLog2e;
  __syncthreads();

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, o[KD][4];
#pragma unroll
  for (int k = 0; k < KD; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) o[k][i] = 0.f;
  const uint32_t ka = (lane & 15) * RB, kx = lane & 7, kc = lane >> 4;
  const uint32_t va = ((lane >> 4) * 8 + (lane & 7)) * RB, vc = lane >> 3 & 1;
  int slot = 0;
  for (int j = jw; j < j1; j += STEP, slot = (slot + 1) % ST) {  // the same trip count for the whole warp
    __syncwarp();  // the tile that the next copies overwrite has been read
    fetch(j + (ST - 1) * STEP, (slot + ST - 1) % ST);
    copy_wait<ST - 1>();
    __syncwarp();
    const uint32_t bits = live & 0xffffu;
    if (bits == 0) continue;
    const uint32_t kt = ring + slot * (2 * TILE), vt = kt + TILE;
    float s[4] = {}, s2[4] = {};
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      uint32_t a[4];
      load_frag(a, kt + ka + (((2 * k + kc) ^ kx) << 4));
      mma<T>(k & 1 ? s2 : s, a, q[k][0], q[k][1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = j + g + 8 * i;
      const bool on = bits >> (g + 8 * i) & 1u;
      const float x0 = (s[2 * i] + s2[2 * i]) * sc + b0[max(-p.R, min(p.R, key - e0))];
      const float x1 = (s[2 * i + 1] + s2[2 * i + 1]) * sc + b1[max(-p.R, min(p.R, key - e1))];
      s[2 * i] = on && ok0 ? x0 : -INFINITY;
      s[2 * i + 1] = on && ok1 ? x1 : -INFINITY;
    }
    // The reference of the exponentials is kLift below the maximum and moves only when a score passes it by kSlack more:
    // P <= 2^15, inside half precision's range, and its small values stay clear of the subnormals.
    const float x0 = fmaxf(s[0], s[2]), x1 = fmaxf(s[1], s[3]);
    if (__any_sync(0xffffffffu, x0 > m0 + (kLift + kSlack) || x1 > m1 + (kLift + kSlack))) {
      float n0 = x0, n1 = x1;
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) {
        n0 = fmaxf(n0, __shfl_xor_sync(0xffffffffu, n0, w));
        n1 = fmaxf(n1, __shfl_xor_sync(0xffffffffu, n1, w));
      }
      n0 = fmaxf(m0, n0 - kLift), n1 = fmaxf(m1, n1 - kLift);
      const float c0 = m0 == n0 ? 1.f : exp2f(m0 - n0), c1 = m1 == n1 ? 1.f : exp2f(m1 - n1);
      m0 = n0, m1 = n1, l0 *= c0, l1 *= c1;
#pragma unroll
      for (int k = 0; k < KD; ++k) o[k][0] *= c0, o[k][1] *= c1, o[k][2] *= c0, o[k][3] *= c1;
    }
    const float f0 = m0 == -INFINITY ? 0.f : m0, f1 = m1 == -INFINITY ? 0.f : m1;  // nothing seen yet: exp2(-inf) = 0
#pragma unroll
    for (int i = 0; i < 2; ++i) s[2 * i] = exp2f(s[2 * i] - f0), s[2 * i + 1] = exp2f(s[2 * i + 1] - f1);
    l0 += s[0] + s[2], l1 += s[1] + s[3];
    uint32_t ph[2], pl[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      split2<T>(s[2 * i], s[2 * i + 1], ph[i], pl[i]);
      ph[i] = transpose8(ph[i]), pl[i] = transpose8(pl[i]);
    }
#pragma unroll
    for (int k = 0; k < KD; ++k) {
      uint32_t a[4];
      load_frag_t(a, vt + va + (((2 * k + vc) ^ kx) << 4));
      mma<T>(o[k], a, ph[0], ph[1]);
      mma<T>(o[k], a, pl[0], pl[1]);
    }
  }
#pragma unroll
  for (int w = 4; w < 32; w <<= 1) l0 += __shfl_xor_sync(0xffffffffu, l0, w), l1 += __shfl_xor_sync(0xffffffffu, l1, w);

  // ---- join the warps ----
  copy_wait<0>();
  __syncthreads();  // the ring and the bias are done with
  constexpr int LD = DP + 4;
  float* so = reinterpret_cast<float*>(smem);  // [NW][8][LD]
  float* sml = so + NW * 8 * LD;               // [NW][8][2]
#pragma unroll
  for (int k = 0; k < KD; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) so[(warp * 8 + r0 + (i & 1)) * LD + 16 * k + g + 8 * (i >> 1)] = o[k][i];
  if (g == 0) {
    sml[2 * (warp * 8 + r0)] = m0, sml[2 * (warp * 8 + r0) + 1] = l0;
    sml[2 * (warp * 8 + r1)] = m1, sml[2 * (warp * 8 + r1) + 1] = l1;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < rows * p.D; x += NW * 32) {
    const int r = x / p.D, d = x - r * p.D;
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, sml[2 * (w * 8 + r)]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float c = exp2f(sml[2 * (w * 8 + r)] - ref);
      L = fmaf(sml[2 * (w * 8 + r) + 1], c, L);
      acc = fmaf(so[(w * 8 + r) * LD + d], c, acc);
    }
    const int h = hk * G + (first + r) / p.Sq, i = (first + r) % p.Sq;
    const int64_t row = ((int64_t)b * p.H + h) * p.Sq + i;
    const int64_t prow = (int64_t)blockIdx.y * p.B * p.H * p.Sq + row;
    if (p.nsplit > 1) {
      p.part_o[prow * p.D + d] = acc;
      if (d == 0) p.part_ml[prow] = make_float2(M, L);
    } else {
      acc = L == 0.f ? 0.f : acc / L;
      row_of<T>(p.o, p.o_s, b, h, i)[d] = from_f32<T>(acc);
      if (p.o32) p.o32[row * p.D + d] = acc;
      if (d == 0 && p.lse) p.lse[row] = log_sum(M, L);
    }
  }
}

int mma_smem(int kd, int G, int R) {
  return std::max(NW * ST * 2 * KT * kd * 32 + std::min(G, 8) * (2 * R + 1) * 4, NW * 8 * (kd * 16 + 6) * 4);
}
template <typename T, int KD>
int launch_mma(const Params& p, int rows, cudaStream_t st) {
  const int smem = mma_smem(KD, p.H / p.Hk, p.R);
  if (int rc = allow_smem<rows_mma_kernel<T, KD>>(smem, "bias_attn_rows")) return rc;
  const int groups = (rows + 7) / 8;
  return launch_pdl("bias_attn_rows", rows_mma_kernel<T, KD>, dim3(p.B * p.Hk * groups, p.nsplit), dim3(NW * 32), smem, st, p,
                    groups);
}
template <typename T>
int mma_by_width(const Params& p, int rows, cudaStream_t st) {
  return p.D <= 64 ? launch_mma<T, 4>(p, rows, st) : launch_mma<T, 8>(p, rows, st);
}

// R: query rows (Sq * G rounded up to a power of two); LPK: lanes per key.
template <int R, int LPK>
__global__ void __launch_bounds__(NW * 32) rows_kernel(const __grid_constant__ Params p, int rows) {
  using T = float;
  constexpr int N = 4, KPW = 32 / LPK, U = R >= 4 ? 2 : 4;
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
      const float4 raw = *reinterpret_cast<const float4*>(row_of<T>(p.q, p.q_s, b, hk * G + r / p.Sq, r % p.Sq) + part * N);
      q[r][0] = raw.x, q[r][1] = raw.y, q[r][2] = raw.z, q[r][3] = raw.w;
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
    float4 kr[U], vr[U];
    bool on[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = j + u * KPW + sub;
      on[u] = key < j1 && (p.mask == nullptr || p.mask[(int64_t)b * p.mask_sb + key] != 0);
      const bool ld = on[u] && has;  // what a masked key holds is not read
      kr[u] = ld ? __ldcs(reinterpret_cast<const float4*>(kb + (int64_t)key * p.k_s[2])) : make_float4(0.f, 0.f, 0.f, 0.f);
      vr[u] = ld ? __ldcs(reinterpret_cast<const float4*>(vb + (int64_t)key * p.v_s[2])) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float s[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float kf[N] = {kr[u].x, kr[u].y, kr[u].z, kr[u].w};
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
      const float vf[N] = {vr[u].x, vr[u].y, vr[u].z, vr[u].w};
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
        o = L == 0.f ? 0.f : o / L;
        row_of<T>(p.o, p.o_s, b, h, i)[d] = o;
        if (p.o32) p.o32[row * p.D + d] = o;
      }
    }
    if (threadIdx.x == 0) {
      if (p.nsplit > 1) p.part_ml[prow] = make_float2(M, L);
      else if (p.lse) p.lse[row] = log_sum(M, L);
    }
    __syncthreads();
  }
}

template <int R, int LPK>
int launch(const Params& p, int rows, cudaStream_t st) {
  constexpr int N = 4, GRP = NW * 32 / LPK;
  const int G = p.H / p.Hk;
  const int smem = std::max(G * (2 * p.R + 1), GRP * (LPK * N + 2)) * 4;
  if (int rc = allow_smem<rows_kernel<R, LPK>>(smem, "bias_attn_rows")) return rc;
  return launch_pdl("bias_attn_rows", rows_kernel<R, LPK>, dim3(p.B * p.Hk, p.nsplit), dim3(NW * 32), smem, st, p, rows);
}

template <int R>
int by_width(const Params& p, int rows, cudaStream_t st) {
  const int lanes = (p.D + 3) / 4;
  if (lanes <= 4) return launch<R, 4>(p, rows, st);
  if (lanes <= 8) return launch<R, 8>(p, rows, st);
  if (lanes <= 16) return launch<R, 16>(p, rows, st);
  return launch<R, 32>(p, rows, st);
}
int by_rows(const Params& p, int rows, cudaStream_t st) {
  if (rows <= 1) return by_width<1>(p, rows, st);
  if (rows <= 2) return by_width<2>(p, rows, st);
  if (rows <= 4) return by_width<4>(p, rows, st);
  return by_width<8>(p, rows, st);
}

}  // namespace

// At most 8 queries (fp32: at most 8 query rows per key/value head), and rows that are whole aligned 16-byte groups. With
// more queries the 128-row tiles win: 8 x 16 heads over 8192 keys of 64 take 90 us here with 16 queries and 127 with 24, 82
// there; with 2 and 4 queries of 4 x 4 key/value heads shared by 8 over 16384 keys of 128, 42 and 75 us here, 160 there.
bool rows_eligible(const b2_bias_attn_args* a) {
  const int64_t es = (int64_t)dtype_size(a->dtype), n = 16 / es;
  auto ok = [&](const void* t, const int64_t* s) {
    return ((uintptr_t)t & 15) == 0 && s[0] % n == 0 && s[1] % n == 0 && s[2] % n == 0;
  };
  return a->Sk >= 1 && a->Sq * (a->dtype == B2_F32 ? a->H / a->Hk : 1) <= 8 && a->D % n == 0 && ok(a->q, a->q_s) && ok(a->k, a->k_s) && ok(a->v, a->v_s);
}

int rows_blocks_per_sm(const b2_bias_attn_args* a) {
  if (a->dtype == B2_F32) return 6;
  const int smem = mma_smem(a->D <= 64 ? 4 : 8, (int)(a->H / a->Hk), a->max_distance);
  return std::max(1, std::min(6, 227 * 1024 / (smem + 1024)));
}

int rows_fwd(const Params& p, int dtype, cudaStream_t st) {
  const int rows = p.Sq * (p.H / p.Hk);
  switch (dtype) {
    case B2_F32: return by_rows(p, rows, st);
    case B2_BF16: return mma_by_width<__nv_bfloat16>(p, rows, st);
    default: return mma_by_width<__half>(p, rows, st);
  }
}

}  // namespace bias_attn
}  // namespace b2
