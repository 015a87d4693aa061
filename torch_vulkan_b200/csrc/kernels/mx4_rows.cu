// y = Q(x) W^T + bias + h b^T for at most 8 rows of x over a frozen MXFP4 weight: bound by reading W once.
//
// Twice an E2M1 value is a whole number (0, 1, 2, 3, 4, 6, 8, 12 with a sign), so a block of 32 products is an exact
// integer sum of dp4a: a lane owns a 32-column block of W (16 bytes, one load) and the same block of each row of x, and
// its sum is scaled once, by a quarter of the two blocks' scales, into an fp32 sum. Four nibbles become four bytes with
// one byte permutation as the table lookup, positive and negative ones apart. Every block of threads quantises x itself
// (it is a few KB), so the call is one launch.
#include "mx4.cuh"
#include "tc_ptx.cuh"

namespace b2 {
namespace {

constexpr int NWARP = 8;
// weight rows per warp at a time, whose loads are in flight together
__host__ __device__ constexpr int rows_per_warp(int M) { return M <= 4 ? 4 : 2; }

struct RowsP {
  const __nv_bfloat16* x;
  int64_t x_ld;
  const uint8_t* codes;
  const uint8_t* scales;
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;
  int64_t out_ld;
  const __nv_bfloat16* h;
  const __nv_bfloat16* lb;
  int64_t h_ld, lb_ld;
  int M, N, K, nblk;  // nblk: 32-column blocks
  int64_t nkb;
  int r;
  int vec;            // rows of x are whole 16-byte groups
};

// Four codes (the low 16 bits of c) -> twice the magnitudes of the positive ones, zeros for the others. A prmt selector
// with bit 3 set gives the byte's sign bit eight times over, which is zero for every entry of this table; with the signs
// flipped it yields the negative ones. (__byte_perm drops that bit.)
__device__ __forceinline__ uint32_t positive4(uint32_t c) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(0x03020100u), "r"(0x0C080604u), "r"(c));
  return r;
}

template <int M>
__global__ void __launch_bounds__(NWARP * 32, 2) mx4_rows_kernel(const __grid_constant__ RowsP p) {
  constexpr int RW = rows_per_warp(M);
  extern __shared__ uint4 sm16[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t cb = (int64_t)p.nblk * 16;
  const int64_t step = (int64_t)gridDim.x * NWARP * RW;
  int64_t n0 = ((int64_t)blockIdx.x * NWARP + warp) * RW;
  // a block of each of the RW rows and its scale; the loads of the next iteration are issued before the work of this one,
  // the first before x is quantised
  uint4 w[RW];
  uint32_t sc[RW];
  auto fetch = [&](int64_t row0, int blk) {
    if (row0 >= p.N || blk >= p.nblk) return;
#pragma unroll
    for (int r = 0; r < RW; ++r) {
      const int64_t n = min(row0 + r, (int64_t)p.N - 1);  // rows past the end repeat the last one
      w[r] = __ldcs(reinterpret_cast<const uint4*>(p.codes + n * cb) + blk);
      sc[r] = p.scales[mx4::scale_at(n, blk, p.nkb)];
    }
  };
  tc::pdl_wait();
  tc::pdl_trigger();
  fetch(n0, lane);
  // x as bytes (twice the E2M1 values) in 32-byte blocks, [M][nblk], and a quarter of its scales
  int* xs = reinterpret_cast<int*>(sm16);
  float* xsc = reinterpret_cast<float*>(xs + M * p.nblk * 8);
  for (int i = threadIdx.x; i < M * p.nblk; i += NWARP * 32) {
    const int m = i / p.nblk, blk = i - m * p.nblk;
    float v[32];
    uint32_t top = 0;
    const int n = m < p.M ? min(32, p.K - blk * 32) : 0;
    const __nv_bfloat16* px = p.x + (int64_t)m * p.x_ld + blk * 32;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (p.vec && q * 8 + 8 <= n) {
        const uint4 raw = *reinterpret_cast<const uint4*>(px + q * 8);
        const __nv_bfloat16* t = reinterpret_cast<const __nv_bfloat16*>(&raw);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[q * 8 + k] = __bfloat162float(t[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[q * 8 + k] = q * 8 + k < n ? __bfloat162float(px[q * 8 + k]) : 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < 32; ++k) top = max(top, mx4::magnitude_bits(v[k]));
    const uint32_t code = mx4::scale_code(top);
    const float inv = mx4::inverse_scale(code);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = code == 255u ? 0.f : v[q * 8 + k] * inv;
      const uint32_t c = mx4::e2m1x8(w);
#pragma unroll
      for (int hlf = 0; hlf < 2; ++hlf) {
        const uint32_t c4 = c >> (16 * hlf);
        xs[i * 8 + q * 2 + hlf] = (int)__vsub4(positive4(c4), positive4(c4 ^ 0x8888u));
      }
    }
    xsc[i] = 0.25f * mx4::e8m0_to_f32(code);
  }
  __syncthreads();

  for (; n0 < p.N; n0 += step) {
    float acc[RW][M];
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m) acc[r][m] = 0.f;
    for (int blk = lane; blk < p.nblk; blk += 32) {
      uint4 cwr[RW];
      uint32_t csc[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) cwr[r] = w[r], csc[r] = sc[r];
      if (blk + 32 < p.nblk) fetch(n0, blk + 32);
      else fetch(n0 + step, lane);
      int xv[M][8];
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const int4* px = reinterpret_cast<const int4*>(xs + (m * p.nblk + blk) * 8);
        *reinterpret_cast<int4*>(&xv[m][0]) = px[0];
        *reinterpret_cast<int4*>(&xv[m][4]) = px[1];
      }
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        const uint32_t cw[4] = {cwr[r].x, cwr[r].y, cwr[r].z, cwr[r].w};
        int s[M], t[M];
#pragma unroll
        for (int m = 0; m < M; ++m) s[m] = t[m] = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const uint32_t c4 = cw[q >> 1] >> (16 * (q & 1));
          const int pos = (int)positive4(c4), neg = (int)positive4(c4 ^ 0x88888888u);
#pragma unroll
          for (int m = 0; m < M; ++m) s[m] = __dp4a(pos, xv[m][q], s[m]), t[m] = __dp4a(neg, xv[m][q], t[m]);
        }
        // the weight's scale first: a sum of 32 products passes fp32's range under the scale of activations above 2^119
        const float ws = mx4::e8m0_to_f32(csc[r]);
#pragma unroll
        for (int m = 0; m < M; ++m) acc[r][m] = fmaf((float)(s[m] - t[m]) * ws, xsc[m * p.nblk + blk], acc[r][m]);
      }
    }
    if (p.r) {  // the LoRA term: two columns of h and b a lane
#pragma unroll
      for (int r = 0; r < RW; ++r) {
        const int64_t n = min(n0 + r, (int64_t)p.N - 1);
        if (2 * lane < p.r) {
          const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p.lb + n * p.lb_ld + 2 * lane));
#pragma unroll
          for (int m = 0; m < M; ++m)
            if (m < p.M) {
              const float2 h = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p.h + (int64_t)m * p.h_ld + 2 * lane));
              acc[r][m] = fmaf(h.x, b.x, fmaf(h.y, b.y, acc[r][m]));
            }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RW; ++r)
#pragma unroll
      for (int m = 0; m < M; ++m) {
        const float s = warp_sum(acc[r][m]);
        const int64_t n = n0 + r;
        if (lane == 0 && m < p.M && n < p.N)
          p.out[(int64_t)m * p.out_ld + n] = __float2bfloat16(s + (p.bias ? __bfloat162float(p.bias[n]) : 0.f));
      }
  }
}

template <int M>
int launch_rows(const RowsP& p, cudaStream_t st) {
  const int smem = M * p.nblk * 36;
  if (int rc = allow_smem<mx4_rows_kernel<M>>(smem, "mx4_rows")) return rc;
  // two blocks to an SM, every block the same number of turns
  const int64_t unit = NWARP * rows_per_warp(M), need = ((int64_t)p.N + unit - 1) / unit;
  const int64_t turns = (need + device_info().sm_count * 2 - 1) / (device_info().sm_count * 2);
  const int grid = (int)((need + turns - 1) / turns);
  return launch_pdl("mx4_rows", mx4_rows_kernel<M>, dim3(grid), dim3(NWARP * 32), smem, st, p);
}

}  // namespace

// At most 8 rows whose bytes and scales fit in half an SM's shared memory. From 4 rows up a large weight is quicker on the
// tensor cores, whose tile takes 128 rows in the time of one. Measured, rows here / there with the quantisation: 2048 -> 18432,
// 1 row 8.1 / 11.4 us, 2 rows 9.5 / 11.4, 4 rows 13.3 / 11.4; 2048 -> 8192, 4 rows 8.2 / 10.2, 8 rows 14.8 / 10.2;
// 2048 -> 2048, 8 rows 7.1 / 9.9.
bool mx4_rows_eligible(const b2_mx4_gemm_args* a) {
  if (a->transpose_w || !a->x || a->M > 8 || a->N >= (1ll << 31) || a->K >= (1ll << 20)) return false;
  const int64_t m = a->M <= 1 ? 1 : a->M <= 2 ? 2 : a->M <= 4 ? 4 : 8;
  if ((a->K + 31) / 32 * 36 * m > 100 * 1024) return false;
  return a->M <= 2 || (double)a->M * (double)a->N * (double)a->K <= 80e6;
}

int mx4_rows(const b2_mx4_gemm_args* a, cudaStream_t st) {
  RowsP p{};
  p.x = (const __nv_bfloat16*)a->x, p.x_ld = a->x_ld;
  p.codes = a->w_codes, p.scales = a->w_scales;
  p.bias = (const __nv_bfloat16*)a->bias;
  p.out = (__nv_bfloat16*)a->out, p.out_ld = a->out_ld;
  p.h = (const __nv_bfloat16*)a->lora_h, p.lb = (const __nv_bfloat16*)a->lora_b, p.h_ld = a->lora_h_ld, p.lb_ld = a->lora_b_ld;
  p.M = (int)a->M, p.N = (int)a->N, p.K = (int)a->K, p.nblk = (int)((a->K + 31) / 32), p.nkb = (a->K + 127) / 128;
  p.r = a->lora_r;
  p.vec = a->x_ld % 8 == 0 && ((uintptr_t)a->x & 15) == 0;
  if (p.M <= 1) return launch_rows<1>(p, st);
  if (p.M <= 2) return launch_rows<2>(p, st);
  if (p.M <= 4) return launch_rows<4>(p, st);
  return launch_rows<8>(p, st);
}

}  // namespace b2
