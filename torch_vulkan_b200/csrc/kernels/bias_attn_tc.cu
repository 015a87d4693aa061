// Relative-position-bias attention on the tensor cores (tcgen05 + TMEM + TMA), bf16 / f16, head dim up to 128 in
// multiples of 8 (columns past D are filled with zeros by the tile loads and clipped by the tile stores).
//
// The bias of a 128-row tile against a key tile depends on key - query alone: it is a slice of one vector of
// 2 max_distance + 509 floats per head in shared memory, which thread = row reads at consecutive addresses across the
// lanes (no bank conflicts); tiles wholly beyond max_distance take one constant instead. The causal mask is part of the
// vector (-inf), the key mask one bit per key from a ballot, and fully hidden tiles at the end are not walked.
#include "bias_attn.cuh"
#include "tc_ptx.cuh"

#include <type_traits>

namespace b2 {

bool make_tmap(CUtensorMap* m, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
               const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle sw);  // gemm_tc.cu

namespace bias_attn {
namespace {

constexpr int kPad = 254;  // a tile that reaches within max_distance spans at most 254 more positions on either side

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (BF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}

__device__ __forceinline__ int vec_len(const Params& p) { return 2 * p.R + 2 * kPad + 1; }
inline int vec_bytes(const Params& p) { return (2 * p.R + 2 * kPad + 1 + 3) / 4 * 16; }

// vec[rel + R + kPad] = bias of head h at rel, log2 units
__device__ __forceinline__ void fill_vec(const Params& p, int h, float* vec, int tid, int n) {
  for (int i = tid; i < vec_len(p); i += n) vec[i] = bias_at(p, h, i - p.R - kPad);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// Whether keys k + lane and k + 32 + lane lie below `end` and are seen, for a ballot later.
struct KeyBytes {
  bool a, b;
};
__device__ __forceinline__ KeyBytes key_bytes(const Params& p, int b, int k, int end) {
  const int j = k + (threadIdx.x & 31);
  const uint8_t* m = p.mask ? p.mask + (int64_t)b * p.mask_sb : nullptr;
  return {j < end && (m == nullptr || m[j] != 0), j + 32 < end && (m == nullptr || m[j + 32] != 0)};
}

// One past the last key below `end` that the mask leaves (every thread of the block; contains block barriers). The whole
// row of the mask is read at once: one trip to memory. slot: shared memory, not in use otherwise.
__device__ __forceinline__ int trim_end(const Params& p, int b, int end, int nthreads, int* slot) {
  if (p.mask == nullptr) return end;
  const uint8_t* m = p.mask + (int64_t)b * p.mask_sb;
  if (threadIdx.x == 0) *slot = 0;
  int last = 0;
#pragma unroll 8
  for (int j = (int)threadIdx.x; j < end; j += nthreads) last = m[j] != 0 ? j + 1 : last;
  __syncthreads();
  last = __reduce_max_sync(0xffffffffu, last);
  if ((threadIdx.x & 31) == 0 && last > 0) atomicMax(slot, last);
  __syncthreads();
  return *slot;
}

// One past the last threshold's distance: where a side's far bucket begins.
__device__ __forceinline__ int far_from(const Params& p) { return p.thr[(p.bidir ? p.nb / 2 : p.nb) - 2]; }

// The bucket whose sum the query side of the backward takes from the others' (see the end of bwd_side), or -1: the far bucket of
// one side where it has more than half of the weight of what the block's middle row sees, exp(bias) for each visible key (v counts
// the far ones; one-sided, keys after the query share bucket 0). So it has a pair, and a bucket that the table all but hides is
// left alone. vec: the head's bias. A whole warp calls it.
__device__ __forceinline__ int big_bucket(const Params& p, const Visible& v, const float* vec, int b, int mid, int end) {
  const int side = p.bidir ? p.nb / 2 : p.nb, far = far_from(p), lane = threadIdx.x & 31;
  const float* at = vec + p.R + kPad;  // centred on relative position 0
  const uint8_t* m = p.mask ? p.mask + (int64_t)b * p.mask_sb : nullptr;
  const float past = v.past > 0 ? at[-far] : -INFINITY, ahead = v.ahead > 0 ? at[p.bidir ? far : 1] : -INFINITY;
  const int first = max(1 - far, -mid), last = min(p.bidir ? far - 1 : p.causal ? 0 : -1, end - 1 - mid);
  const float top = fmaxf(past, ahead);
  if (top == -INFINITY) return -1;
  float near = 0.f;  // infinite where the far keys weigh next to nothing beside it
#pragma unroll 8
  for (int r = first + lane; r <= last; r += 32) near += m == nullptr || m[mid + r] != 0 ? ex2(at[r] - top) : 0.f;
  const float wp = v.past * ex2(past - top), wa = v.ahead * ex2(ahead - top), half = 0.5f * (warp_sum(near) + wp + wa);
  return wp > half ? side - 1 : wa > half ? (p.bidir ? p.nb - 1 : 0) : -1;
}

// A warp's 32 rows of O (TMEM, relative to the maximum m) and their earlier part (relative to run_m): in TMEM columns of its own
// at D = 64, else in memory, column by column, `rows` floats each (the rows that exist), in the place that the finished rows will
// take. OUT: the sum joins the earlier part; else it goes back to O.
template <int D, bool OUT>
__device__ __forceinline__ void add_run(uint32_t t_o, uint32_t t_sum, float* part, bool first, float run_m, float m, int rows,
                                        int dims) {
  const int lane = threadIdx.x & 31;
  const bool on = lane < rows;
  const float w = first ? 0.f : run_m == m ? 1.f : ex2(run_m - m);
#pragma unroll 1
  for (int c = 0; c < D / 16; ++c) {
    uint32_t o[16], y[16];
    float* at = part + c * 16 * rows + lane;
    __syncwarp();
    if (D == 64) {
      if (!first) tc::tmem_ld16(t_sum + c * 16, y);
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) y[e] = !first && on && c * 16 + e < dims ? __float_as_uint(at[e * rows]) : 0u;
    }
    tc::tmem_ld16(t_o + c * 16, o);
    tc::tmem_wait_ld();
    tc::reg_fence16(o);
    if (D == 64) tc::reg_fence16(y);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float x = first ? __uint_as_float(o[e]) : fmaf(__uint_as_float(y[e]), w, __uint_as_float(o[e]));
      o[e] = __float_as_uint(x);
      if (OUT && D != 64 && on && c * 16 + e < dims) at[e * rows] = x;
    }
    if (!OUT || D == 64) tc::tmem_st16((OUT ? t_sum : t_o) + c * 16, o);
  }
  tc::tmem_wait_st();
  __syncwarp();
}

// ==================================================================================================
// forward: a block owns 128 queries of a head and walks the keys in tiles of 64 with two score buffers, so that the next
// scores are multiplied while a softmax runs. Two blocks share an SM (256 TMEM columns, half of the shared memory each), so
// that one's set-up, softmax and output run beside the other's. The softmax bounds it: 1800 cycles a tile, 800 of them
// exponentials of two warps on one scheduler (scores are always ready when they are asked for). 16 heads x 4096 x 4096 x 64:
// 135 us, for a backward (below) 170. One block to an SM with two softmax groups took 24.5 us against 20.8 at B4 H16 S512
// D64 and 110 against 94 at B8 H16 S1024 D128 (padded); tiles of 128 with one score buffer 165 us against 151; two threads
// to a row, 32 columns each, 213 against 174 (for a backward).
// ==================================================================================================
template <int D>
struct Fwd {
  static constexpr int BQ = 128, BK = 64, DCH = D / 64;
  static constexpr int Q_BYTES = BQ * D * 2, KV_BYTES = BK * D * 2;
  static constexpr int NK = D == 64 ? 4 : 2, NV = NK;  // K / V ring depths: what two blocks fit
  static constexpr int OFF_Q = 0, OFF_K = Q_BYTES, OFF_V = OFF_K + NK * KV_BYTES, OFF_BAR = OFF_V + NV * KV_BYTES;
  static constexpr int OFF_VEC = OFF_BAR + 256;
  static constexpr int THREADS = 192;
  // PREC: tiles whose P V is summed before the sum leaves the accumulator, to columns of its own where TMEM has them; through
  // memory a move takes 3 us, so fewer are made (every 8 tiles: 256 us, every 16: 220)
  static constexpr int RUN = D == 64 ? 8 : 16;
  static constexpr uint32_t T_S = 0, T_O = 128, T_SUM = 192, TMEM_COLS = 256;  // T_SUM: D = 64
};

// PREC (o32 wanted, for a backward): P enters the product as two 16-bit numbers, P = hi + lo, so that O is good to about
// 2^-17 before its rounding. delta = rowsum(dO O) is made from it, and dS = P (dP - delta) cancels over a row: with P
// rounded once, the bias gradient (a sum of dS over many rows) keeps errors of a few 1e-3 of itself. The tensor core also
// truncates each of its sums towards zero: after 4096 keys (512 of them) O is 8.3e-6 of itself short, and the gradient of a far
// bucket adds that up over all rows (1e-5 of it). So every RUN tiles the sum joins a sum kept in fp32 elsewhere and the next one
// starts from zero: 1.1e-6 short at D = 64 (2.0e-6 at D = 128), gradient 1e-6 to 2.5e-6 off; 9 % more time and, through memory,
// 22 % (16 heads x 4096 x 4096).
template <int D, bool BF16, bool PREC>
__global__ void __launch_bounds__(192, 2)
    bias_fwd_tc(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ Params p) {
  using C = Fwd<D>;
  constexpr int NK = C::NK, NV = C::NV;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bar;
  uint64_t* k_full = bar + 1;         // [NK]
  uint64_t* k_empty = k_full + NK;    // [NK]
  uint64_t* v_full = k_empty + NK;    // [NV]
  uint64_t* v_empty = v_full + NV;    // [NV]
  uint64_t* s_full = v_empty + NV;    // [2] S of tile t in buffer t & 1 of TMEM
  uint64_t* p_full = s_full + 2;      // [2] P of tile t in TMEM over S
  uint64_t* o_upd = p_full + 2;       // [2] P V of the last tile but one, of the last
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_upd + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(o_upd + 3);
  float* vec = reinterpret_cast<float*>(smem + C::OFF_VEC);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // causal: the tiles with the most keys start first
  const int qt = p.causal ? (int)(gridDim.x - 1 - blockIdx.x) : (int)blockIdx.x;
  const int q0 = qt * C::BQ;
  const int b = (int)blockIdx.y / p.H, h = (int)blockIdx.y % p.H, hk = h / (p.H / p.Hk);

  if (threadIdx.x == 0) {
    tc::mbar_init(q_full, 1);
    for (int i = 0; i < NK; ++i) tc::mbar_init(&k_full[i], 1), tc::mbar_init(&k_empty[i], 1);
    for (int i = 0; i < NV; ++i) tc::mbar_init(&v_full[i], 1), tc::mbar_init(&v_empty[i], 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(&s_full[i], 1), tc::mbar_init(&p_full[i], 4), tc::mbar_init(&o_upd[i], 1);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  tc::pdl_wait();
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, C::TMEM_COLS);
    tc::tmem_relinquish();
  }
  const int end = trim_end(p, b, key_end(p, min(q0 + C::BQ, p.Sq) - 1), C::THREADS, reinterpret_cast<int*>(vec));
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  tc::pdl_trigger();
  const int ntiles = (end + C::BK - 1) / C::BK;
  const int per = (ntiles + p.nsplit - 1) / p.nsplit;
  const int t0 = (int)blockIdx.z * per;
  const int n = max(0, min(per, ntiles - t0));  // tiles of this block: t0 .. t0 + n

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      // ---------------- producer ----------------
      bool ok = true;
      tc::mbar_arrive_expect_tx(q_full, C::Q_BYTES);
      for (int c = 0; c < C::DCH; ++c) tc::tma_load_4d(smem + C::OFF_Q + c * (C::BQ * 128), &tmQ, q_full, c * 64, q0, h, b);
      int issued_k[NK] = {}, issued_v[NV] = {};
      for (int t = 0; t < n; ++t) {
        const int s = t % NK, v = t % NV, k0 = (t0 + t) * C::BK;
        if (!tc::mbar_wait(&k_empty[s], (uint32_t)((t / NK) & 1) ^ 1, p.err) || *abort_flag) { ok = false; break; }
        tc::mbar_arrive_expect_tx(&k_full[s], C::KV_BYTES);
        for (int c = 0; c < C::DCH; ++c)
          tc::tma_load_4d(smem + C::OFF_K + s * C::KV_BYTES + c * (C::BK * 128), &tmK, &k_full[s], c * 64, k0, hk, b);
        issued_k[s]++;
        if (!tc::mbar_wait(&v_empty[v], (uint32_t)((t / NV) & 1) ^ 1, p.err) || *abort_flag) { ok = false; break; }
        tc::mbar_arrive_expect_tx(&v_full[v], C::KV_BYTES);
        for (int c = 0; c < C::DCH; ++c)
          tc::tma_load_4d(smem + C::OFF_V + v * C::KV_BYTES + c * (C::BK * 128), &tmV, &v_full[v], c * 64, k0, hk, b);
        issued_v[v]++;
      }
      if (!ok) {
        *abort_flag = 1;
        tc::mbar_wait(q_full, 0, nullptr);
        for (int s = 0; s < NK; ++s)
          if (issued_k[s]) tc::mbar_wait(&k_full[s], (uint32_t)((issued_k[s] - 1) & 1), nullptr);
        for (int s = 0; s < NV; ++s)
          if (issued_v[s]) tc::mbar_wait(&v_full[s], (uint32_t)((issued_v[s] - 1) & 1), nullptr);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && n > 0) {
      // ---------------- MMA issuer: S_t = Q K_t^T; O += P_t V_t with P_t read from TMEM; then S_t+2 over P_t's columns
      // (MMAs of one thread execute in order), while the softmax warps are at S_t+1 ----------------
      constexpr uint32_t IDESC_S = tc::idesc_f16(128, C::BK, BF16, false, false);
      constexpr uint32_t IDESC_O = tc::idesc_f16(128, D, BF16, false, true);
      const tc::SDesc qd = tc::sdesc_parts(tc::smem_u32(smem + C::OFF_Q), 16, 1024);
      bool ok = tc::mbar_wait(q_full, 0, p.err);
      auto issue_s = [&](int t) -> bool {
        const int ks = t % NK;
        if (!tc::mbar_wait(&k_full[ks], (uint32_t)((t / NK) & 1), p.err)) return false;
        tc::tc_fence_after();
        const tc::SDesc kd = tc::sdesc_parts(tc::smem_u32(smem + C::OFF_K + ks * C::KV_BYTES), 16, 1024);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          tc::mma_f16_ss(tbase + C::T_S + (t & 1) * C::BK, tc::sdesc_at(qd, (k >> 2) * (C::BQ * 128) + (k & 3) * 32),
                         tc::sdesc_at(kd, (k >> 2) * (C::BK * 128) + (k & 3) * 32), IDESC_S, k > 0 ? 1u : 0u);
        }
        tc::mma_commit(&s_full[t & 1]);
        tc::mma_commit(&k_empty[ks]);
        return true;
      };
      if (ok) ok = issue_s(0);
      if (ok && n > 1) ok = issue_s(1);
      for (int t = 0; t < n && ok; ++t) {
        const int vs = t % NV;
        if (!tc::mbar_wait(&p_full[t & 1], (uint32_t)((t >> 1) & 1), p.err) ||
            !tc::mbar_wait(&v_full[vs], (uint32_t)((t / NV) & 1), p.err)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const tc::SDesc vd = tc::sdesc_parts(tc::smem_u32(smem + C::OFF_V + vs * C::KV_BYTES), C::BK * 128, 1024);
#pragma unroll
        for (int k = 0; k < C::BK / 16; ++k)
          tc::mma_f16_ts(tbase + C::T_O, tbase + C::T_S + (t & 1) * C::BK + k * 8, tc::sdesc_at(vd, k * 2048), IDESC_O, (k > 0 || (PREC ? t % C::RUN != 0 : t > 0)) ? 1u : 0u);
        if (PREC) {
#pragma unroll
          for (int k = 0; k < C::BK / 16; ++k)
            tc::mma_f16_ts(tbase + C::T_O, tbase + C::T_S + (t & 1) * C::BK + 32 + k * 8, tc::sdesc_at(vd, k * 2048), IDESC_O, 1u);
        }
        if (t >= n - 2) tc::mma_commit(&o_upd[t - (n - 2)]);
        tc::mma_commit(&v_empty[vs]);
        if (t + 2 < n && !issue_s(t + 2)) ok = false;
      }
      if (!ok) *abort_flag = 1;
    }
  } else {
    // ---------------- softmax warps: thread = query row ----------------
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t t_o = tbase + C::T_O;
    const float sl2 = p.scale * kLog2e;
    const float2 sl22 = make_float2(sl2, sl2);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    fill_vec(p, h, vec, (int)threadIdx.x - 64, 128);  // while the first tiles are loaded and multiplied
    tc::named_bar_sync(1, 128);
    // PREC: this warp's rows of o32 (of the split's partial output), and the maximum that what lies there is relative to
    const int run_rows = max(0, min(32, p.Sq - q0 - quarter * 32));
    float* run_o = nullptr;
    float run_m = 0.f;
    if (PREC) {
      const int64_t row = (int64_t)blockIdx.y * p.Sq + q0 + quarter * 32;
      run_o = p.nsplit > 1 ? p.part_o + ((int64_t)blockIdx.z * p.B * p.H * p.Sq + row) * p.D : p.o32 + row * p.D;
    }
    const float far_lo = vec[0], far_hi = vec[vec_len(p) - 1];  // the bias beyond max_distance
    const int wholes = p.mask == nullptr ? end / C::BK - t0 : 0;  // tiles without a key to leave out
    KeyBytes kb = key_bytes(p, b, t0 * C::BK, end);
    for (int t = 0; t < n; ++t) {
      const int k0 = (t0 + t) * C::BK;
      const uint32_t t_s = tbase + C::T_S + (t & 1) * C::BK;
      uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
      if (t >= wholes) {
        bits[0] = __ballot_sync(0xffffffffu, kb.a), bits[1] = __ballot_sync(0xffffffffu, kb.b);
        kb = key_bytes(p, b, k0 + C::BK, end);  // the next tile's, on their way during this one
      } else if (t + 1 == wholes) {
        kb = key_bytes(p, b, k0 + C::BK, end);
      }
      const bool full = (bits[0] & bits[1]) == 0xffffffffu;
      if (!tc::mbar_wait(&s_full[t & 1], (uint32_t)((t >> 1) & 1), p.err) || *abort_flag) {
        ok = false;
        break;
      }
      tc::tc_fence_after();
      uint32_t sr[C::BK];
      __syncwarp();
#pragma unroll
      for (int c = 0; c < C::BK / 32; ++c) tc::tmem_ld32(t_s + c * 32 + lane_off, sr + 32 * c);
      tc::tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < C::BK / 32; ++c) tc::reg_fence32(sr + 32 * c);
      // bias: x = s * scale_log2 + bias. rel of column 0 against this tile's first row
      const int rel0 = k0 - q0 - p.q_off;
      const bool near = rel0 - 127 < p.R && rel0 + (C::BK - 1) > -p.R;
      float cst = 0.f;
      if (near) {
        const float* bv = vec + (rel0 - r + p.R + kPad);
#pragma unroll
        for (int e = 0; e < C::BK; e += 2) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(sr[e]), __uint_as_float(sr[e + 1])), sl22,
                                      make_float2(bv[e], bv[e + 1]));
          sr[e] = __float_as_uint(x.x), sr[e + 1] = __float_as_uint(x.y);
        }
      } else {
        cst = rel0 > 0 ? far_hi : far_lo;
      }
      if (!full) {
#pragma unroll
        for (int e = 0; e < C::BK; ++e)
          if (!((bits[e >> 5] >> (e & 31)) & 1u)) sr[e] = __float_as_uint(-INFINITY);
      }
      float mx8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) mx8[e] = __uint_as_float(sr[e]);
#pragma unroll
      for (int e = 8; e < C::BK - 8; e += 16)
#pragma unroll
        for (int i = 0; i < 8; ++i) mx8[i] = max3(mx8[i], __uint_as_float(sr[e + i]), __uint_as_float(sr[e + 8 + i]));
#pragma unroll
      for (int i = 0; i < 8; ++i) mx8[i] = fmaxf(mx8[i], __uint_as_float(sr[C::BK - 8 + i]));
      const float mx = fmaxf(max3(mx8[0], mx8[1], mx8[2]), max3(max3(mx8[3], mx8[4], mx8[5]), mx8[6], mx8[7]));
      const float mul = near ? 1.f : sl2;  // scale > 0
      const float m_blk = fmaf(mx, mul, cst);
      // keep the old maximum unless the new one is more than 2^8 larger
      const bool need = m_blk > m + 8.f || (m == -INFINITY && m_blk > -INFINITY);
      const bool fresh = PREC && t % C::RUN == 0;  // this tile's P V starts a new sum
      const bool moves = __any_sync(0xffffffffu, need);
      if (t > 0 && (moves || fresh)) {
        // O is read: the last tile's P V is in it once the next scores are there (MMAs execute in order)
        if (!__all_sync(0xffffffffu, t + 1 < n ? tc::mbar_wait(&s_full[(t + 1) & 1], (uint32_t)(((t + 1) >> 1) & 1), p.err)
                                               : tc::mbar_wait(&o_upd[0], 0, p.err))) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
      }
      if (PREC && fresh && t > 0) {
        add_run<D, true>(t_o + lane_off, tbase + C::T_SUM + lane_off, run_o, t == C::RUN, run_m, m, run_rows, p.D);
        run_m = m;
      }
      if (moves) {
        float alpha = 1.f;
        if (need) {
          alpha = (m == -INFINITY) ? 0.f : ex2(m - m_blk);
          m = m_blk;
        }
        l *= alpha;
        if (t > 0 && !fresh) {  // O moves to the new maximum
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t orow[16];
            tc::tmem_ld16(t_o + c * 16 + lane_off, orow);
            tc::tmem_wait_ld();
            tc::reg_fence16(orow);
#pragma unroll
            for (int e = 0; e < 16; ++e) orow[e] = __float_as_uint(__uint_as_float(orow[e]) * alpha);
            tc::tmem_st16(t_o + c * 16 + lane_off, orow);
          }
        }
      }
      const float nmv = (m == -INFINITY) ? -INFINITY : cst - m;  // nothing seen yet: exp2(-inf) = 0
      const float2 nm = make_float2(nmv, nmv), mul2 = make_float2(mul, mul);
      float2 rs4[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
      {
        uint32_t w[C::BK / 2];
#pragma unroll
        for (int i = 0; i < C::BK / 2; ++i) {
          const float2 x = __ffma2_rn(make_float2(__uint_as_float(sr[2 * i]), __uint_as_float(sr[2 * i + 1])), mul2, nm);
          const float2 e2 = make_float2(ex2(x.x), ex2(x.y));
          rs4[i & 3] = __fadd2_rn(rs4[i & 3], e2);
          w[i] = pack2<BF16>(e2.x, e2.y);
          if (PREC) {  // what the rounding left
            const float2 hi = unpack2<BF16>(w[i]);
            sr[2 * i] = pack2<BF16>(e2.x - hi.x, e2.y - hi.y);
          }
        }
        tc::tmem_st32(t_s + lane_off, w);
        if (PREC) {
#pragma unroll
          for (int i = 0; i < C::BK / 2; ++i) w[i] = sr[2 * i];
          tc::tmem_st32(t_s + 32 + lane_off, w);
        }
      }
      const float2 rs2 = __fadd2_rn(__fadd2_rn(rs4[0], rs4[1]), __fadd2_rn(rs4[2], rs4[3]));
      l += rs2.x + rs2.y;
      if (!full && (p.mask != nullptr || end < p.Sk)) {
        // keys that the mask or the causal rule hides may hold anything, and 0 * NaN is NaN in the P V product: clear their
        // rows of V (past Sk the load has put zeros)
        if (!tc::mbar_wait(&v_full[t % NV], (uint32_t)((t / NV) & 1), p.err)) { ok = false; break; }
        if (!((bits[quarter & 1] >> lane) & 1u)) {  // warps 0 and 1 clear one half of a row, 2 and 3 the other
#pragma unroll
          for (int c = 0; c < C::DCH; ++c) {
            uint4* row = reinterpret_cast<uint4*>(smem + C::OFF_V + (t % NV) * C::KV_BYTES + c * (C::BK * 128) + (r & 63) * 128 +
                                                  (quarter >> 1) * 64);
#pragma unroll
            for (int i = 0; i < 4; ++i) row[i] = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        tc::fence_async_shared();
        __syncwarp();
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&p_full[t & 1]);
    }
    // ---------------- epilogue ----------------
    if (ok && n > 0 && !tc::mbar_wait(&o_upd[1], 0, p.err)) ok = false;
    if (ok && !*abort_flag) {
      tc::tc_fence_after();
      const bool split = p.nsplit > 1;
      const float inv = split ? 1.f : inverse_sum(l);
      const int qrow = q0 + r;
      const int64_t row = (int64_t)blockIdx.y * p.Sq + qrow;
      const int64_t prow = (int64_t)blockIdx.z * p.B * p.H * p.Sq + row;
      if (PREC && n > C::RUN) add_run<D, false>(t_o + lane_off, tbase + C::T_SUM + lane_off, run_o, false, run_m, m, run_rows, p.D);
      uint8_t* stg = smem + C::OFF_K + (warp - 2) * (D / 32) * 2048;  // every MMA that read K is done
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        if (c * 32 >= p.D) break;
        float v[32];
        {
          uint32_t o[32];
          __syncwarp();
          if (n > 0) {
            tc::tmem_ld32(tbase + C::T_O + c * 32 + lane_off, o);
            tc::tmem_wait_ld();
            tc::reg_fence32(o);
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = n > 0 ? __uint_as_float(o[e]) * inv : 0.f;
        }
        if ((split || PREC) && qrow < p.Sq) {
          float* po = (split ? p.part_o + prow * p.D : p.o32 + row * p.D) + c * 32;
#pragma unroll
          for (int e = 0; e < 32; e += 4)
            if (c * 32 + e < p.D) *reinterpret_cast<float4*>(po + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
        }
        if (split) continue;
        // O rows leave through a per-warp staging tile, one 32 x 32 box per tile store
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = pack2<BF16>(v[2 * e], v[2 * e + 1]);
        uint8_t* buf = stg + c * 2048;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<uint4*>(buf + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) =
              make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        tc::fence_async_shared();
        __syncwarp();
        if (lane == 0 && q0 + quarter * 32 < p.Sq) {
          tc::tma_store_4d(&tmO, buf, c * 32, q0 + quarter * 32, h, b);
          tc::bulk_commit();
        }
      }
      if (qrow < p.Sq) {
        if (split) p.part_ml[prow] = make_float2(m, l);
        else if (p.lse) p.lse[row] = l == 0.f ? -INFINITY : (m + __log2f(l)) * kLn2;
      }
      if (lane == 0) tc::bulk_wait0();
    } else {
      *abort_flag = 1;
    }
  }
  __syncwarp();  // warps 0 and 1 arrive diverged; the block barrier is an aligned one
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tbase, C::TMEM_COLS);
  }
}

// ==================================================================================================
// backward: the same walk with the two sides in either place. The fixed side's two operands X1, X2 (128 rows) stay in
// shared memory, the walked side's Y1, Y2 come in tiles of NT rows:
//   KEYS = false  X = Q, dO (a block owns 128 queries), Y = K, V:   dQ += dS K, and the bias gradient
//   KEYS = true   X = K, V (a block owns 128 keys),    Y = Q, dO:   dK += dS^T Q, dV += P^T dO, over every query head
//                                                                   that shares the key/value head
// S = X1 Y1^T and dP = X2 Y2^T are recomputed on both sides (7 products instead of 5), which leaves every gradient one
// owner: no atomics, no accumulator in memory, the same bits on every run. Two teams of eight warps take the tiles in turn;
// in a team, two warps share a lane quarter and split its columns. P and dS (16 bits) replace the scores a warp has read and
// are the A operands of the gradient MMAs, 8 columns per 16 of the reduction at any place. At D = 64 TMEM holds three tiles,
// so that the MMAs of one run while both teams work (4 x 16 heads x 512 x 512: 60 us, with two tiles of 96 columns 67). The two
// issuing threads bound it: one among element-wise warps takes 80 to 140 cycles for a product of 48 (16 heads x 4096 x
// 4096: 366 us at D = 64, 464 at 128). Eight element-wise warps, half as many, took 357 us instead of 285 for the key side alone.
// ==================================================================================================
template <int D, bool KEYS>
struct Bwd {
  static constexpr int BX = 128, DCH = D / 64;
  static constexpr int NT = 64;                  // walked rows per tile
  static constexpr int NB = D == 64 ? 3 : 2;     // tiles of scores in TMEM: what it holds beside the sums
  static constexpr int HC = NT / 2;                        // columns of a tile per warp
  static constexpr int X_BYTES = BX * D * 2, Y_BYTES = NT * D * 2;
  static constexpr int LD_BYTES = KEYS ? NT * 8 : 0;       // (-lse log2 e, -delta) of the walked queries
  static constexpr int STAGE = 2 * Y_BYTES + (LD_BYTES + 1023) / 1024 * 1024;
  // ring depth: a stage is freed by the gradient MMAs of its tile, and its next load takes about a microsecond from there.
  // Two stages at D = 128 put that latency into every tile (612 us for the key side alone at 16 heads x 4096 x 4096 x 128)
  static constexpr int NS = D == 64 ? 7 : (KEYS ? 4 : 3);
  static constexpr int OFF_X = 0, OFF_Y = 2 * X_BYTES, OFF_BAR = OFF_Y + NS * STAGE, OFF_VEC = OFF_BAR + 256;
  static constexpr int EW = 512, THREADS = 64 + EW + 32;   // element-wise threads; producer, two MMA issuers
  static constexpr uint32_t T_S = 0, T_DP = NT, T_BUF = 2 * NT, T_ACC = NB * T_BUF, TMEM_COLS = 512;
  static constexpr uint32_t T_ACC2 = T_ACC + D;  // KEYS: dV at T_ACC, dK behind it
  static_assert(NB * T_BUF + (KEYS ? 2 * D : D) <= 512, "TMEM columns");
  // columns of the A operand's 16-deep step k, counted from the scores' first column
  static __device__ __forceinline__ constexpr uint32_t a_col(int k) { return k < HC / 16 ? k * 8 : HC + (k - HC / 16) * 8; }
};

// Adds the diagonal sums of a 32 x 16 block (rows = lanes, v = this lane's 16 columns) to arr[clamp(rel + column - row)],
// where arr is centred on relative position 0 and spans -R .. R. Running sums travel up the lanes by one per column: the
// sum that lane l holds at column e belongs to the diagonal e - l; the one that has passed lane 31 is complete and is put
// aside. Positions beyond +-R share a slot: those lanes are added up first.
__device__ __forceinline__ void add_at(float* arr, int pos, float x, bool on, int R, int lane) {
  const bool hi = on && pos > R, lo = on && pos < -R;
  if (__any_sync(0xffffffffu, hi || lo)) {
    const float sh = warp_sum(hi ? x : 0.f), sl = warp_sum(lo ? x : 0.f);
    if (lane == 0) arr[R] += sh, arr[-R] += sl;
    __syncwarp();
  }
  if (on && !hi && !lo) arr[pos] += x;
  __syncwarp();
}
__device__ __forceinline__ void add_diagonals(const float* v, float* arr, int rel, int R, float* scratch, int lane) {
  float a = v[0];
  const int from = (lane + 31) & 31;
#pragma unroll
  for (int e = 1; e < 16; ++e) {
    float t = __shfl_sync(0xffffffffu, a, from);
    if (lane == 0) {
      scratch[e - 1] = t;
      t = 0.f;
    }
    a = t + v[e];
  }
  __syncwarp();
  add_at(arr, rel + 15 - lane, a, true, R, lane);
  add_at(arr, rel + lane - 31, lane < 15 ? scratch[lane] : 0.f, lane < 15, R, lane);
}

// f16: the exponent of the factor that dS is rounded under, as large as it can be: |dS| <= |dP| + |delta| <= 2 max |dO_i| max |V_j|,
// which it brings to 2^13.5 .. 2^15 for the rows of a key/value head. Without it the gradients of a loss that was not scaled lose
// bits: dq of 1000 keys is 0.37 % off at dO = 2^-12 and 5.6 % at 2^-16, where the rounding to f16 alone leaves 0.04 % and 0.5 %.
__device__ __forceinline__ int ds_up(const Params& p, int b, int hk) {
  const uint2 n = *reinterpret_cast<const uint2*>(p.norms + 2 * ((int64_t)b * p.Hk + hk));
  const int exps = (int)(n.x >> 23) + (int)(n.y >> 23) - 2 * 127;  // of the two squared norms together
  return n.x && n.y ? max(-40, min(60, 13 - ((exps + 1) >> 1))) : 0;
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// block: index among the blocks of this side, xtiles of them per head.
template <int D, bool BF16, bool KEYS>
__device__ __forceinline__ void bwd_side(const CUtensorMap& tmX1, const CUtensorMap& tmX2, const CUtensorMap& tmY1,
                                         const CUtensorMap& tmY2, const CUtensorMap& tmG1, const CUtensorMap& tmG2,
                                         const Params& p, const float2* __restrict__ lsed, int sq_pad, int block, int xtiles) {
  using C = Bwd<D, KEYS>;
  constexpr int NS = C::NS, NT = C::NT, HC = C::HC, NB = C::NB;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* x_full = bar;
  uint64_t* y_full = bar + 1;          // [NS]
  uint64_t* y_empty = y_full + NS;     // [NS]
  uint64_t* sd_full = y_empty + NS;    // [NB] S and dP of tile t in buffer t % NB
  uint64_t* pd_full = sd_full + NB;     // [NB] P / dS of tile t in TMEM (one arrival per warp of the team)
  uint64_t* acc_full = pd_full + NB;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(acc_full + 2);
  volatile int* big_slot = abort_flag + 1;  // !KEYS: big_bucket of this block, and one past its last key
  const int vlen4 = (vec_len(p) + 3) / 4 * 4, dlen = (2 * p.R + 1 + 3) / 4 * 4;
  float* vec = reinterpret_cast<float*>(smem + C::OFF_VEC);  // KEYS: one per team (the head changes along the walk)
  float* darr = vec + vlen4;                                 // !KEYS: diagonal sums, one array per warp
  float* dscr = darr + 16 * dlen;                            // !KEYS: 16 floats per warp; at the end the buckets' sums

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = KEYS ? p.Hk : p.H, G = p.H / p.Hk;
  // causal: the query tiles with the most keys come first; the key tiles with the most queries already do
  const int bh = block / xtiles, xi = block - bh * xtiles;
  const int xt = (!KEYS && p.causal) ? xtiles - 1 - xi : xi;
  const int x0 = xt * C::BX;
  const int b = bh / heads, hx = bh % heads;

  if (threadIdx.x == 0) {
    tc::mbar_init(x_full, 1);
    for (int i = 0; i < NS; ++i) tc::mbar_init(&y_full[i], 1), tc::mbar_init(&y_empty[i], 2);
    for (int i = 0; i < NB; ++i) tc::mbar_init(&sd_full[i], 2), tc::mbar_init(&pd_full[i], 8);
    tc::mbar_init(acc_full, 2);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  tc::pdl_wait();
  if (warp == 1) {
    tc::tmem_alloc(tmem_slot, C::TMEM_COLS);
    tc::tmem_relinquish();
  }
  Visible seen = {};
  const int mid = x0 + min(C::BX, p.Sq - x0) / 2 + p.q_off;  // !KEYS: the position of the block's middle row
  int first = 0, tiles, end = p.Sk;  // tiles first .. first + tiles of every walked head; !KEYS: one past the last key
  if (KEYS) {
    const int any = p.mask == nullptr ||
                    __syncthreads_or((int)threadIdx.x < C::BX && x0 + (int)threadIdx.x < p.Sk &&
                                     p.mask[(int64_t)b * p.mask_sb + x0 + threadIdx.x] != 0);
    const int nt = (p.Sq + NT - 1) / NT;
    if (p.causal) first = (int)min((int64_t)nt, max((int64_t)0, (int64_t)x0 - p.q_off) / NT);
    tiles = any ? nt - first : 0;
  } else {
    seen = visible_keys(p, b, key_end(p, min(x0 + C::BX, p.Sq) - 1), mid - far_from(p), p.bidir ? mid + far_from(p) : mid,
                        C::THREADS, reinterpret_cast<int*>(vec));
    end = seen.last;
    if (threadIdx.x == 0) big_slot[1] = end;
    tiles = (end + NT - 1) / NT;
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  tc::pdl_trigger();
  const int n = KEYS ? tiles * G : tiles;

  if (warp == 0) {
    if (lane == 0 && n > 0) {
      // ---------------- producer ----------------
      tc::mbar_arrive_expect_tx(x_full, 2 * C::X_BYTES);
      for (int c = 0; c < C::DCH; ++c) {
        tc::tma_load_4d(smem + C::OFF_X + c * (C::BX * 128), &tmX1, x_full, c * 64, x0, hx, b);
        tc::tma_load_4d(smem + C::OFF_X + C::X_BYTES + c * (C::BX * 128), &tmX2, x_full, c * 64, x0, hx, b);
      }
      int issued[NS] = {};
      bool ok = true;
      for (int t = 0; t < n; ++t) {
        const int s = t % NS;
        const int gi = KEYS ? t / tiles : 0;
        const int hy = KEYS ? hx * G + gi : hx / G;
        const int y0 = KEYS ? (first + t - gi * tiles) * NT : t * NT;
        if (!tc::mbar_wait(&y_empty[s], (uint32_t)((t / NS) & 1) ^ 1, p.err) || *abort_flag) { ok = false; break; }
        uint8_t* st = smem + C::OFF_Y + s * C::STAGE;
        tc::mbar_arrive_expect_tx(&y_full[s], 2 * C::Y_BYTES + C::LD_BYTES);
        for (int c = 0; c < C::DCH; ++c) {
          tc::tma_load_4d(st + c * (NT * 128), &tmY1, &y_full[s], c * 64, y0, hy, b);
          tc::tma_load_4d(st + C::Y_BYTES + c * (NT * 128), &tmY2, &y_full[s], c * 64, y0, hy, b);
        }
        if (KEYS) tc::bulk_load(st + 2 * C::Y_BYTES, lsed + ((int64_t)b * p.H + hy) * sq_pad + y0, C::LD_BYTES, &y_full[s]);
        issued[s]++;
      }
      if (!ok) {
        *abort_flag = 1;
        tc::mbar_wait(x_full, 0, nullptr);
        for (int s = 0; s < NS; ++s)
          if (issued[s]) tc::mbar_wait(&y_full[s], (uint32_t)((issued[s] - 1) & 1), nullptr);
      }
    }
  } else if (warp == 1 || warp == C::THREADS / 32 - 1) {
    if (lane == 0 && n > 0) {
      // ---------------- MMA issuers: one for S and what is made of the columns it leaves (dV or dQ), one for dP and dK.
      // The MMAs of one thread execute in order, so a tile's gradient has read its P or dS before the next scores land there.
      // An issuing thread shares its scheduler with four element-wise warps and gets few of its slots: with a single one the
      // backward of 16 heads x 4096 x 4096 x 128 took 560 us instead of 473. Loads by one of the two instead of their own warp:
      // 620 us ----------------
      constexpr uint32_t IDESC_S = tc::idesc_f16(128, NT, BF16, false, false);
      constexpr uint32_t IDESC_G = tc::idesc_f16(128, D, BF16, false, true);
      const bool second = warp != 1;
      const tc::SDesc x = tc::sdesc_parts(tc::smem_u32(smem + C::OFF_X + (second ? C::X_BYTES : 0)), 16, 1024);
      const uint32_t y_of = second ? C::Y_BYTES : 0, g_of = second ? 0 : (KEYS ? C::Y_BYTES : 0);
      const uint32_t t_sd = tbase + (second ? C::T_DP : C::T_S), t_acc = tbase + (second ? C::T_ACC2 : C::T_ACC);
      bool ok = tc::mbar_wait(x_full, 0, p.err);
      auto issue_sd = [&](int t) -> bool {
        const int s = t % NS;
        if (!tc::mbar_wait(&y_full[s], (uint32_t)((t / NS) & 1), p.err)) return false;
        tc::tc_fence_after();
        const tc::SDesc y = tc::sdesc_parts(tc::smem_u32(smem + C::OFF_Y + s * C::STAGE) + y_of, 16, 1024);
        const uint32_t dst = t_sd + (t % NB) * C::T_BUF;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc::mma_f16_ss(dst, tc::sdesc_at(x, (k >> 2) * (C::BX * 128) + (k & 3) * 32),
                         tc::sdesc_at(y, (k >> 2) * (NT * 128) + (k & 3) * 32), IDESC_S, k > 0 ? 1u : 0u);
        tc::mma_commit(&sd_full[t % NB]);
        return true;
      };
      for (int t = 0; t < NB && t < n && ok; ++t) ok = issue_sd(t);
      for (int t = 0; t < n && ok; ++t) {
        const int s = t % NS;
        if (!tc::mbar_wait(&pd_full[t % NB], (uint32_t)((t / NB) & 1), p.err)) { ok = false; break; }
        tc::tc_fence_after();
        if (KEYS || !second) {  // KEYS: dV += P^T dO and dK += dS^T Q; else dQ += dS K
          const tc::SDesc y = tc::sdesc_parts(tc::smem_u32(smem + C::OFF_Y + s * C::STAGE) + g_of, NT * 128, 1024);
          const uint32_t src = t_sd + (t % NB) * C::T_BUF;
#pragma unroll
          for (int k = 0; k < NT / 16; ++k)
            tc::mma_f16_ts(t_acc, src + C::a_col(k), tc::sdesc_at(y, k * 2048), IDESC_G, k > 0 || t > 0 ? 1u : 0u);
        }
        tc::mma_commit(&y_empty[s]);
        if (t + NB < n && !issue_sd(t + NB)) ok = false;
      }
      if (ok) tc::mma_commit(acc_full);
      else *abort_flag = 1;
    }
  } else {
    // ---------------- element-wise warps: thread = row of the fixed side, half of the tile's columns ----------------
    const int w16 = warp - 2;                        // 0..15
    const int g = w16 >> 3, hh = (w16 >> 2) & 1, quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int tt = hh * 128 + r;                     // thread of the team, 0..255
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const uint32_t buf0 = tbase + hh * HC + lane_off;  // this warp's columns of S (and, + T_DP, of dP) in the first buffer
    const float sl2 = p.scale * kLog2e;
    const float2 sl22 = make_float2(sl2, sl2);
    // f16: P carries a factor of 2^8 (in its bias) so that 1 / Sk stays clear of the subnormals; dS carries 2^ds_up
    constexpr float PUP = BF16 ? 0.f : 8.f;
    constexpr float PDOWN = BF16 ? 1.f : 1.f / 256.f;
    float ds_mul = PDOWN;
    float* myvec = KEYS ? vec + g * vlen4 : vec;
    float* mydarr = darr + w16 * dlen + p.R;         // centred on relative position 0
    float* myscr = dscr + w16 * 16;
    float nL = 0.f, nd = 0.f;  // !KEYS: -(lse log2 e) and -delta of this row
    if (!KEYS) {  // while the first tiles are loaded and multiplied
      const float2 ld = lsed[((int64_t)b * p.H + hx) * sq_pad + x0 + r];
      nL = ld.x, nd = ld.y;
      fill_vec(p, hx, vec, (int)threadIdx.x - 64, C::EW);
      if (p.dtab)
        for (int i = (int)threadIdx.x - 64; i < 16 * dlen; i += C::EW) darr[i] = 0.f;
      tc::named_bar_sync(1, C::EW);
      if (w16 == 15 && p.dtab) {  // of the team whose first tile comes later
        const int big = big_bucket(p, seen, vec, b, mid, end);
        if (lane == 0) *big_slot = big;
      }
      if (sees_one(p, x0 + r, seen.first, seen.second) && isfinite(nL + nd)) nL = -INFINITY;  // dS = 0; a NaN goes its way
      if (!BF16) nL += (float)ds_up(p, b, hx / G);  // P times 2^ds_up: this side needs it for dS alone
    }
    float far_lo = 0.f, far_hi = 0.f;
    int cur = -1;  // KEYS: the head whose bias is in myvec
    bool ok = true;
    float b_lo = 0.f, b_hi = 0.f;  // the bias beyond max_distance
    if (!KEYS) b_lo = vec[0], b_hi = vec[vec_len(p) - 1];
    const int wholes = KEYS || p.mask != nullptr ? 0 : end / NT;  // !KEYS: tiles without a key to leave out
    KeyBytes keys = {true, true};
    if (!KEYS) keys = key_bytes(p, b, g * NT + hh * HC, end);
    int gi = 0, yi = g;  // tile t is tile yi of the walked head gi
    for (int t = g; t < n; t += 2, yi += 2) {
      if (KEYS)
        while (yi >= tiles) yi -= tiles, ++gi;
      const int y0 = (KEYS ? first + yi : t) * NT;
      if (KEYS && gi != cur) {
        tc::named_bar_sync(2 + g, 256);  // nobody still reads the last head's
        for (int i = tt; i < vec_len(p); i += 256) myvec[i] = bias_at(p, hx * G + gi, i - p.R - kPad) + PUP;
        tc::named_bar_sync(2 + g, 256);
        cur = gi;
        b_lo = myvec[0], b_hi = myvec[vec_len(p) - 1];
        if (!BF16) ds_mul = PDOWN * exp2i(ds_up(p, b, hx));
      }
      // after a wait that ran out the tiles are still counted off, so that the team meets at the barriers above
      if (!ok) continue;
      uint64_t bits = ~0ull;  // !KEYS: one bit per column of this warp
      bool full = true;
      if (!KEYS && t >= wholes) {
        const uint32_t b0 = __ballot_sync(0xffffffffu, keys.a), b1 = __ballot_sync(0xffffffffu, keys.b);
        bits = (uint64_t)b0 | ((uint64_t)b1 << 32);
        full = (~bits & ((1ull << HC) - 1)) == 0;
      }
      if (!KEYS && t + 2 >= wholes) keys = key_bytes(p, b, y0 + 2 * NT + hh * HC, big_slot[1]);  // this team's next tile's, on their way
      // relative position of column 0 against row 0, and how it moves: -row + column (queries own the rows) or +row - column
      const int rel0 = KEYS ? x0 - y0 - p.q_off : y0 - x0 - p.q_off;
      const bool near = KEYS ? (rel0 - (NT - 1) < p.R && rel0 + 127 > -p.R) : (rel0 - 127 < p.R && rel0 + (NT - 1) > -p.R);
      const float* bv = myvec + (rel0 + (KEYS ? r - hh * HC : hh * HC - r) + p.R + kPad);
      const float cst = near ? 0.f : (rel0 > 0 ? b_hi : b_lo);
      const int bi = t % NB;
      const uint32_t buf = buf0 + bi * C::T_BUF;
      if (!tc::mbar_wait(&sd_full[bi], (uint32_t)((t / NB) & 1), p.err) || *abort_flag ||
          (KEYS && !tc::mbar_wait(&y_full[t % NS], (uint32_t)((t / NS) & 1), p.err))) {
        ok = false;
        continue;
      }
      tc::tc_fence_after();
      __syncwarp();
      const float4* ld4 = reinterpret_cast<const float4*>(smem + C::OFF_Y + (t % NS) * C::STAGE + 2 * C::Y_BYTES) + hh * (HC / 2);
      // one straight piece of code for each kind of tile
      auto walk = [&](auto near_c, auto mask_c) {
        constexpr bool NEAR = decltype(near_c)::value, MASK = decltype(mask_c)::value;
        const float2 row_off = make_float2(nL + cst, nL + cst), row_del = make_float2(nd, nd);
#pragma unroll
        for (int c = 0; c < HC / 16; ++c) {
          uint32_t sv[16], dp[16];
          tc::tmem_ld16(buf + C::T_S + c * 16, sv);
          tc::tmem_ld16(buf + C::T_DP + c * 16, dp);
          tc::tmem_wait_ld();
          tc::reg_fence16(sv);
          tc::reg_fence16(dp);
          uint32_t wp[8], wd[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int col = c * 16 + 2 * e;
            float2 off = row_off, del = row_del;
            if (KEYS) {
              const float4 L = ld4[col >> 1];
              off = make_float2(L.x, L.z), del = make_float2(L.y, L.w);
              off = __fadd2_rn(off, NEAR ? make_float2(bv[-col], bv[-col - 1]) : make_float2(cst, cst));
            } else if (NEAR) {
              off = __fadd2_rn(off, make_float2(bv[col], bv[col + 1]));
            }
            const float2 x = __ffma2_rn(make_float2(__uint_as_float(sv[2 * e]), __uint_as_float(sv[2 * e + 1])), sl22, off);
            const float2 pr = make_float2(ex2(x.x), ex2(x.y));
            float2 dd = __fadd2_rn(make_float2(__uint_as_float(dp[2 * e]), __uint_as_float(dp[2 * e + 1])), del);
            if (KEYS && !BF16) dd = __fmul2_rn(dd, make_float2(ds_mul, ds_mul));
            float2 ds = __fmul2_rn(pr, dd);
            if (MASK) {
              if (!((bits >> col) & 1ull)) ds.x = 0.f;
              if (!((bits >> (col + 1)) & 1ull)) ds.y = 0.f;
            }
            if (KEYS) wp[e] = pack2<BF16>(pr.x, pr.y);
            wd[e] = pack2<BF16>(ds.x, ds.y);
            if (!KEYS) sv[2 * e] = __float_as_uint(ds.x), sv[2 * e + 1] = __float_as_uint(ds.y);
          }
          // P over S, dS over dP (KEYS) or over S: 8 columns whose scores this warp has read
          if (KEYS) {
            tc::tmem_st8(buf + C::T_S + c * 8, wp);
            tc::tmem_st8(buf + C::T_DP + c * 8, wd);
          } else {
            tc::tmem_st8(buf + C::T_S + c * 8, wd);
            if (p.dtab) {
              const float* dsv = reinterpret_cast<const float*>(sv);
              if (NEAR) {
                add_diagonals(dsv, mydarr, rel0 + hh * HC + c * 16 - quarter * 32, p.R, myscr, lane);
              } else {
                float s = 0.f;
#pragma unroll
                for (int e = 0; e < 16; ++e) s += dsv[e];
                if (rel0 > 0) far_hi += s;
                else far_lo += s;
              }
            }
          }
        }
      };
      using yes = std::true_type;
      using no = std::false_type;
      if (near) {
        if (KEYS || full) walk(yes{}, no{});
        else walk(yes{}, std::integral_constant<bool, !KEYS>{});
      } else {
        if (KEYS || full) walk(no{}, no{});
        else walk(no{}, std::integral_constant<bool, !KEYS>{});
      }
      if (!KEYS && !full) {
        // hidden keys may hold anything, and 0 * NaN is NaN in the dS K product: clear their rows of K
        for (int i = lane; i < HC; i += 32)
          if (!((bits >> i) & 1ull) && quarter < 2 * C::DCH) {
            // the four warps of this column half share the work: 64 bytes of a row each
            uint4* row = reinterpret_cast<uint4*>(smem + C::OFF_Y + (t % NS) * C::STAGE + (quarter >> 1) * (NT * 128) +
                                                  (hh * HC + i) * 128 + (quarter & 1) * 64);
#pragma unroll
            for (int j = 0; j < 4; ++j) row[j] = make_uint4(0u, 0u, 0u, 0u);
          }
        tc::fence_async_shared();
      }
      tc::tmem_wait_st();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&pd_full[bi]);
    }
    const float ds_down = BF16 ? 1.f : exp2i(-ds_up(p, b, KEYS ? hx : hx / G));
    if (!KEYS && p.dtab) {
      // this warp's far tiles join the ends of its array; then the arrays are added and cut into buckets
      const float lo = warp_sum(far_lo), hi = warp_sum(far_hi);
      if (lane == 0) mydarr[-p.R] += lo, mydarr[p.R] += hi;
      tc::named_bar_sync(1, C::EW);
      for (int i = (int)threadIdx.x - 64; i < 2 * p.R + 1; i += C::EW) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += darr[w * dlen + i];
        vec[i] = s;  // the bias itself is no longer needed
      }
      tc::named_bar_sync(1, C::EW);
      // bucket i of a side holds the distances [thr[i - 1], thr[i]), the last one all beyond
      for (int bk = w16; bk < p.nb; bk += 16) {
        const int side = p.bidir ? p.nb / 2 : p.nb;
        const bool pos = p.bidir && bk >= side;
        const int i = pos ? bk - side : bk;
        int d0 = i == 0 ? 0 : (int)p.thr[i - 1];
        const int d1 = i == side - 1 ? p.R + 1 : (int)p.thr[i];
        float s = 0.f;
        if (pos) {
          d0 = max(d0, 1);
          for (int d = d0 + lane; d < d1; d += 32) s += vec[p.R + d];
        } else {
          for (int d = d0 + lane; d < d1; d += 32) s += vec[p.R - d];
          if (!p.bidir && i == 0)  // one-sided: keys after the query share bucket 0
            for (int d = 1 + lane; d <= p.R; d += 32) s += vec[p.R + d];
        }
        s = warp_sum(s);
        if (lane == 0) dscr[bk] = s * ds_down;
      }
      tc::named_bar_sync(1, C::EW);
      // A row of dS adds up to zero over its keys. Where most of the block's weight lies in one bucket (beyond the last threshold on
      // one side) that bucket's sum is minus the others': what an error of delta leaves in a bucket goes with the share of P there.
      // A NaN or infinity that only the bucket itself has stays
      if (w16 == 0) {
        const int big = *big_slot;
        float rest = 0.f;
        for (int i = lane; i < p.nb; i += 32) rest += i == big ? 0.f : dscr[i];
        rest = warp_sum(rest);
        for (int i = lane; i < p.nb; i += 32) p.dtab[(int64_t)block * p.nb + i] = i == big ? 0.f * dscr[i] - rest : dscr[i];
      }
    }
    // ---------------- epilogue: a warp writes 32 rows x 32 columns of a gradient at a time ----------------
    if (ok && n > 0) ok = tc::mbar_wait(acc_full, 0, p.err);
    if (ok && !*abort_flag) {
      tc::tc_fence_after();
      const int rows = KEYS ? p.Sk : p.Sq;
      // a hidden key's row of the sums holds whatever its K and V gave: its gradient is zero
      const bool live = !KEYS || (x0 + r < key_end(p, p.Sq - 1) && (p.mask == nullptr || p.mask[(int64_t)b * p.mask_sb + x0 + r] != 0));
      constexpr int CH = D / 32, JOBS = (KEYS ? 2 : 1) * CH;
      // staging in the idle Y ring: every MMA that read it is done
      uint8_t* stg = smem + C::OFF_Y + w16 * 4096;
      int use = 0;
      for (int job = w16 >> 2; job < JOBS; job += 4, ++use) {
        const int which = job / CH, c = job % CH;  // KEYS: dV, then dK
        const bool wanted = KEYS ? (which ? p.dk != nullptr : p.dv != nullptr) : p.dq != nullptr;
        if (!wanted) continue;
        const float mul = KEYS && !which ? PDOWN : p.scale * ds_down;
        const CUtensorMap* tm = which ? &tmG2 : &tmG1;
        uint32_t v[32], w[16];
        __syncwarp();
        if (n > 0) {
          tc::tmem_ld32(tbase + (which ? C::T_ACC2 : C::T_ACC) + c * 32 + lane_off, v);
          tc::tmem_wait_ld();
          tc::reg_fence32(v);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
          w[e] = n > 0 && live ? pack2<BF16>(__uint_as_float(v[2 * e]) * mul, __uint_as_float(v[2 * e + 1]) * mul) : 0u;
        uint8_t* sb = stg + (use & 1) * 2048;  // at most two jobs a warp
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<uint4*>(sb + lane * 64 + ((e ^ ((lane >> 1) & 3)) << 4)) =
              make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
        tc::fence_async_shared();
        __syncwarp();
        if (lane == 0 && x0 + quarter * 32 < rows && c * 32 < p.D) {
          tc::tma_store_4d(tm, sb, c * 32, x0 + quarter * 32, hx, b);
          tc::bulk_commit();
        }
      }
      if (lane == 0) tc::bulk_wait0();
    } else {
      *abort_flag = 1;
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tbase, C::TMEM_COLS);
  }
}

// Both sides in one launch: the key blocks, whose walks are the longer ones, start first and the query blocks fill the SMs
// that they leave.
struct BwdMaps {
  CUtensorMap qx, gx, ky, vy, dq;  // query side: boxes of Q, dO it owns, of K, V it walks, and dQ
  CUtensorMap kx, vx, qy, gy, dv, dk;
};
template <int D, bool BF16>
__global__ void __launch_bounds__(608, 1)
    bias_bwd_tc(const __grid_constant__ BwdMaps m, const __grid_constant__ Params p, const float2* __restrict__ lsed, int sq_pad,
                int key_blocks, int key_tiles, int query_tiles) {
  if ((int)blockIdx.x < key_blocks)
    bwd_side<D, BF16, true>(m.kx, m.vx, m.qy, m.gy, m.dv, m.dk, p, lsed, sq_pad, blockIdx.x, key_tiles);
  else
    bwd_side<D, BF16, false>(m.qx, m.gx, m.ky, m.vy, m.dq, m.dq, p, lsed, sq_pad, (int)blockIdx.x - key_blocks, query_tiles);
}

// Sum over eight lanes (a row of the prepared tensors).
__device__ __forceinline__ float sum8(float s) {
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  return s + __shfl_xor_sync(0xffffffffu, s, 4);
}
// The block's largest finite value of x >= 0, into *at: floats without a sign are ordered as their bits, and a maximum does not
// depend on the order.
__device__ __forceinline__ void block_max(float x, uint32_t* at) {
  __shared__ uint32_t top[8];
  const uint32_t m = __reduce_max_sync(0xffffffffu, x <= 3.4e38f ? __float_as_uint(x) : 0u);
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t t = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t = max(t, top[i]);
    if (t) atomicMax(at, t);
  }
}

// lsed[bh][q] = (-lse log2 e, -sum_d dO O) for q < Sq, (-inf, 0) for padding and for rows without a key: exp2(x - inf) = 0.
// Eight lanes a row, 16-byte loads, 32 rows of one head a block. With p.norms (f16), the blocks from row_blocks on take the rows
// of V that some query sees, and both kinds record their largest norm.
template <typename T>
__global__ void __launch_bounds__(256) bias_bwd_prep(const __grid_constant__ Params p, float2* __restrict__ lsed, int sq_pad,
                                                     int64_t row_blocks) {
  tc::pdl_wait();
  tc::pdl_trigger();
  const int part = threadIdx.x & 7, r = threadIdx.x >> 3;
  if ((int64_t)blockIdx.x >= row_blocks) {
    const int tiles = (p.Sk + 31) / 32;
    const int64_t vb = blockIdx.x - row_blocks, bh = vb / tiles;
    const int j = (int)(vb - bh * tiles) * 32 + r, b = (int)(bh / p.Hk);
    float s = 0.f;
    if (j < key_end(p, p.Sq - 1) && (p.mask == nullptr || p.mask[(int64_t)b * p.mask_sb + j] != 0)) {
      const T* v = row_of<T>(p.v, p.v_s, b, (int)(bh % p.Hk), j);
      for (int d = part * 8; d < p.D; d += 64) {
        const uint4 raw = *reinterpret_cast<const uint4*>(v + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = to_f32<T>(reinterpret_cast<const T*>(&raw)[i]);
          s = fmaf(x, x, s);
        }
      }
    }
    block_max(sum8(s), p.norms + 2 * bh + 1);
    return;
  }
  const int64_t idx = (int64_t)blockIdx.x * 32 + r, bh = idx / sq_pad;
  const int q = (int)(idx - bh * sq_pad);
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  float s = 0.f, g2 = 0.f;
  if (q < p.Sq) {
    const T* o = row_of<T>((const void*)p.o, p.o_s, b, h, q);
    const T* g = row_of<T>(p.d_o, p.do_s, b, h, q);
    for (int d = part * 8; d < p.D; d += 64) {
      const uint4 b4 = *reinterpret_cast<const uint4*>(g + d);
      const T* c = reinterpret_cast<const T*>(&b4);
      float a[8];
      if (p.o32) {
        const float4* f = reinterpret_cast<const float4*>(p.o32 + (bh * p.Sq + q) * p.D + d);
        const float4 lo = f[0], hi = f[1];
        a[0] = lo.x, a[1] = lo.y, a[2] = lo.z, a[3] = lo.w, a[4] = hi.x, a[5] = hi.y, a[6] = hi.z, a[7] = hi.w;
      } else {
        const uint4 a4 = *reinterpret_cast<const uint4*>(o + d);
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = to_f32<T>(reinterpret_cast<const T*>(&a4)[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(a[i], to_f32<T>(c[i]), s);
      if (std::is_same<T, __half>::value) {
#pragma unroll
        for (int i = 0; i < 8; ++i) g2 = fmaf(to_f32<T>(c[i]), to_f32<T>(c[i]), g2);
      }
    }
  }
  s = sum8(s);
  const float lse = q < p.Sq ? p.lse[bh * p.Sq + q] : -INFINITY;
  if (part == 0) lsed[idx] = lse == -INFINITY ? make_float2(-INFINITY, 0.f) : make_float2(-lse * kLog2e, -s);
  if (std::is_same<T, __half>::value) {
    g2 = sum8(g2);
    block_max(lse == -INFINITY ? 0.f : g2, p.norms + 2 * ((int64_t)b * p.Hk + h / (p.H / p.Hk)));
  }
}

bool bhsd_map(CUtensorMap* m, const void* base, const int64_t* s3, int64_t B, int64_t H, int64_t S, int64_t D, bool bf16,
              uint32_t box_rows, uint32_t box_inner = 64, CUtensorMapSwizzle sw = CU_TENSOR_MAP_SWIZZLE_128B) {
  uint64_t dims[4] = {(uint64_t)D, (uint64_t)S, (uint64_t)H, (uint64_t)B};
  uint64_t strides[3] = {(uint64_t)s3[2] * 2, (uint64_t)s3[1] * 2, (uint64_t)s3[0] * 2};
  // dimensions of size 1: any valid stride
  if (S == 1) strides[0] = (uint64_t)((D + 7) / 8 * 8) * 2;
  if (H == 1) strides[1] = strides[0] * (uint64_t)S;
  if (B == 1) strides[2] = strides[1] * (uint64_t)H;
  uint32_t box[4] = {box_inner, box_rows, 1, 1};
  return make_tmap(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, base, dims, strides, box, sw);
}
bool store_map(CUtensorMap* m, void* base, const int64_t* s3, int64_t B, int64_t H, int64_t S, int64_t D, bool bf16) {
  memset(m, 0, sizeof(*m));
  return base == nullptr || bhsd_map(m, base, s3, B, H, S, D, bf16, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B);
}

// 16-byte aligned rows with positive strides below 2^40 bytes
bool layout_ok(const void* t, const int64_t* s, int64_t B, int64_t H, int64_t S) {
  auto ok = [](int64_t v) { return v > 0 && v % 8 == 0 && v < (1ll << 38); };
  return ((uintptr_t)t & 15) == 0 && (S <= 1 || ok(s[2])) && (H <= 1 || ok(s[1])) && (B <= 1 || ok(s[0]));
}

template <int D, bool BF16, bool PREC>
int fwd_t(const Params& p, cudaStream_t st) {
  using C = Fwd<D>;
  const int smem = C::OFF_VEC + vec_bytes(p) + 1024;
  auto kern = bias_fwd_tc<D, BF16, PREC>;
  if (int rc = allow_smem<bias_fwd_tc<D, BF16, PREC>>(smem, "bias_attn_fwd_tc")) return rc;
  CUtensorMap tq, tk, tv, to;
  if (!bhsd_map(&tq, p.q, p.q_s, p.B, p.H, p.Sq, p.D, BF16, 128) || !bhsd_map(&tk, p.k, p.k_s, p.B, p.Hk, p.Sk, p.D, BF16, C::BK) ||
      !bhsd_map(&tv, p.v, p.v_s, p.B, p.Hk, p.Sk, p.D, BF16, C::BK) || !store_map(&to, p.o, p.o_s, p.B, p.H, p.Sq, p.D, BF16))
    return fail(B2_ERR_ARG, "bias_attn_fwd: tensor map rejected");
  dim3 grid((p.Sq + 127) / 128, p.B * p.H, p.nsplit);
  return launch_pdl("bias_attn_fwd_tc", kern, grid, dim3(C::THREADS), smem, st, tq, tk, tv, to, p);
}

template <int D, bool KEYS>
int bwd_smem(const Params& p) {
  const int vb = vec_bytes(p);
  const int db = (2 * p.R + 1 + 3) / 4 * 16;
  return Bwd<D, KEYS>::OFF_VEC + (KEYS ? 2 * vb : vb + (p.dtab ? 16 * db + 16 * 64 : 0)) + 1024;
}

template <int D, bool BF16>
int bwd_t(const Params& p, float2* lsed, int sq_pad, cudaStream_t st) {
  using T = typename std::conditional<BF16, __nv_bfloat16, __half>::type;
  static_assert(kTcPad % 32 == 0, "whole blocks of rows per head");
  const int64_t row_blocks = (int64_t)p.B * p.H * (sq_pad / 32), v_blocks = BF16 ? 0 : (int64_t)p.B * p.Hk * ((p.Sk + 31) / 32);
  if (row_blocks + v_blocks >= (1ll << 31)) return fail(B2_ERR_ARG, "bias_attn_bwd: too many rows");
  if (int rc = launch_pdl("bias_attn_bwd_prep", bias_bwd_prep<T>, dim3((unsigned)(row_blocks + v_blocks)), dim3(256), 0, st, p,
                          lsed, sq_pad, row_blocks))
    return rc;
  using Q = Bwd<D, false>;
  using K = Bwd<D, true>;
  static_assert(Q::THREADS == K::THREADS, "one launch for both sides");
  const int ktiles = (p.Sk + 127) / 128, qtiles = (p.Sq + 127) / 128;
  const int64_t kblocks = p.dk || p.dv ? (int64_t)p.B * p.Hk * ktiles : 0;
  const int64_t qblocks = p.dq || p.dtab ? (int64_t)p.B * p.H * qtiles : 0;
  if (kblocks + qblocks == 0) return 0;
  if (kblocks + qblocks >= (1ll << 31)) return fail(B2_ERR_ARG, "bias_attn_bwd: too many tiles");
  const int smem = std::max(kblocks ? bwd_smem<D, true>(p) : 0, qblocks ? bwd_smem<D, false>(p) : 0);
  if (int rc = allow_smem<bias_bwd_tc<D, BF16>>(smem, "bias_attn_bwd_tc")) return rc;
  BwdMaps m;
  auto in = [&](CUtensorMap* t, const void* base, const int64_t* s, int heads, int len, uint32_t box) {
    return bhsd_map(t, base, s, p.B, heads, len, p.D, BF16, box);
  };
  if (!in(&m.qx, p.q, p.q_s, p.H, p.Sq, 128) || !in(&m.gx, p.d_o, p.do_s, p.H, p.Sq, 128) ||
      !in(&m.ky, p.k, p.k_s, p.Hk, p.Sk, Q::NT) || !in(&m.vy, p.v, p.v_s, p.Hk, p.Sk, Q::NT) ||
      !in(&m.kx, p.k, p.k_s, p.Hk, p.Sk, 128) || !in(&m.vx, p.v, p.v_s, p.Hk, p.Sk, 128) ||
      !in(&m.qy, p.q, p.q_s, p.H, p.Sq, K::NT) || !in(&m.gy, p.d_o, p.do_s, p.H, p.Sq, K::NT) ||
      !store_map(&m.dq, p.dq, p.dq_s, p.B, p.H, p.Sq, p.D, BF16) || !store_map(&m.dk, p.dk, p.dk_s, p.B, p.Hk, p.Sk, p.D, BF16) ||
      !store_map(&m.dv, p.dv, p.dv_s, p.B, p.Hk, p.Sk, p.D, BF16))
    return fail(B2_ERR_ARG, "bias_attn_bwd: tensor map rejected");
  return launch_pdl("bias_attn_bwd_tc", bias_bwd_tc<D, BF16>, dim3((unsigned)(kblocks + qblocks)), dim3(K::THREADS), smem, st, m, p,
                    (const float2*)lsed, sq_pad, (int)kblocks, ktiles, qtiles);
}

}  // namespace

// What the tensor-core kernels take: 16-bit tensors with D a multiple of 8 (TMA rows are whole 16-byte groups), aligned
// rows, and a positive scale (the running maximum is taken before scaling). scale * log2 e must be finite.
bool tc_fwd_eligible(const b2_bias_attn_args* a) {
  if (a->dtype != B2_BF16 && a->dtype != B2_F16) return false;
  if (!device_info().tcgen05 || a->Sk < 1 || a->D % 8 || !(a->scale > 0.f) || !(a->scale < 1e30f)) return false;
  return layout_ok(a->q, a->q_s, a->B, a->H, a->Sq) && layout_ok(a->k, a->k_s, a->B, a->Hk, a->Sk) &&
         layout_ok(a->v, a->v_s, a->B, a->Hk, a->Sk) && (a->o == nullptr || layout_ok(a->o, a->o_s, a->B, a->H, a->Sq));
}

bool tc_bwd_eligible(const b2_bias_attn_args* a) {
  if (!tc_fwd_eligible(a)) return false;
  if (!layout_ok(a->d_o, a->do_s, a->B, a->H, a->Sq) || (a->dq && !layout_ok(a->dq, a->dq_s, a->B, a->H, a->Sq)) ||
      (a->dk && !layout_ok(a->dk, a->dk_s, a->B, a->Hk, a->Sk)) || (a->dv && !layout_ok(a->dv, a->dv_s, a->B, a->Hk, a->Sk)))
    return false;
  // the bias gradient of a long max_distance at wide heads does not fit beside the tiles
  Params p{};
  p.R = a->max_distance, p.dtab = a->dtable;
  const int need = a->D <= 64 ? bwd_smem<64, false>(p) : bwd_smem<128, false>(p);
  return need <= device_info().smem_optin;
}

template <bool BF16>
int fwd_d(const Params& p, cudaStream_t st) {
  if (p.D <= 64) return p.o32 ? fwd_t<64, BF16, true>(p, st) : fwd_t<64, BF16, false>(p, st);
  return p.o32 ? fwd_t<128, BF16, true>(p, st) : fwd_t<128, BF16, false>(p, st);
}
int tc_fwd(const Params& p, bool bf16, cudaStream_t st) { return bf16 ? fwd_d<true>(p, st) : fwd_d<false>(p, st); }

int tc_bwd(const Params& p, bool bf16, float2* lsed, int sq_pad, cudaStream_t st) {
  if (p.D <= 64) return bf16 ? bwd_t<64, true>(p, lsed, sq_pad, st) : bwd_t<64, false>(p, lsed, sq_pad, st);
  return bf16 ? bwd_t<128, true>(p, lsed, sq_pad, st) : bwd_t<128, false>(p, lsed, sq_pad, st);
}

}  // namespace bias_attn
}  // namespace b2
