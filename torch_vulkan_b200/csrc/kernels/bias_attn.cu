// Entry points of the relative-position-bias attention: argument checks, the bucket thresholds, the choice of kernel,
// and the small kernels both paths share (joining key splits, delta, the last sum of the bias gradient).
#include <cmath>

#include "bias_attn.cuh"
#include "tc_ptx.cuh"

namespace b2 {
namespace bias_attn {
namespace {

// One-sided thresholds: the bucket of a distance n is the number of thresholds <= n. With L = nb - first buckets
// spaced by their logarithm, bucket first + s starts at the smallest n with (n / first)^L >= (max_distance / first)^s.
// The comparison is made on logarithms in extended precision; equal powers differ there by a few 1e-19, unequal ones
// by more than 1e-12 over the whole accepted range of parameters.
int thresholds(int nb, int max_distance, uint16_t* thr) {
  const int first = nb / 2, L = nb - first;
  int n = 0;
  for (int i = 1; i < first; ++i) thr[n++] = (uint16_t)i;
  int d = first;
  for (int s = 0; s < L; ++s) {
    const long double want = (long double)s * logl((long double)max_distance / first);
    while (d < max_distance && (long double)L * logl((long double)d / first) < want - 1e-13L) ++d;
    thr[n++] = (uint16_t)d;
  }
  return n;
}

bool bucket_args_ok(int32_t nb, int32_t max_distance, int32_t bidir) {
  const int side = bidir ? nb / 2 : nb;
  return nb <= B2_BIAS_MAX_BUCKETS && side >= 2 && !(bidir && nb % 2) && max_distance > side / 2 &&
         max_distance <= B2_BIAS_MAX_DISTANCE;
}

// O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over the key splits, one block of four warps per query row: each warp
// adds up every fourth split, four of them in flight, and the four sums are added in order.
template <typename T>
__global__ void __launch_bounds__(128) combine_kernel(const __grid_constant__ Params p) {
  __shared__ float so[4][128], sl[4];
  const int64_t nrow = (int64_t)p.B * p.H * p.Sq;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  tc::pdl_wait();
  float M = -INFINITY;
  for (int s = lane; s < p.nsplit; s += 32) M = fmaxf(M, p.part_ml[s * nrow + row].x);
  M = warp_max(M);
  const float ref = M == -INFINITY ? 0.f : M;
  float acc[4] = {}, l = 0.f;
#pragma unroll 4
  for (int s = warp; s < p.nsplit; s += 4) {
    const float2 ml = p.part_ml[s * nrow + row];
    const float w = exp2f(ml.x - ref);
    l = fmaf(ml.y, w, l);
    const float* po = p.part_o + (s * nrow + row) * p.D;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float o = lane + 32 * i < p.D ? po[lane + 32 * i] : 0.f;
      acc[i] = fmaf(o, w, acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) so[warp][lane + 32 * i] = acc[i];
  if (lane == 0) sl[warp] = l;
  __syncthreads();
  const float L = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const float inv = inverse_sum(L);
  const int64_t i = row % p.Sq, bh = row / p.Sq;
  const int d = threadIdx.x;
  if (d < p.D) {
    const float o = ((so[0][d] + so[1][d]) + (so[2][d] + so[3][d])) * inv;
    row_of<T>(p.o, p.o_s, (int)(bh / p.H), (int)(bh % p.H), i)[d] = from_f32<T>(o);
    if (p.o32) p.o32[row * p.D + d] = o;
  }
  if (d == 0 && p.lse) p.lse[row] = log_sum(M, L);
}

// delta[row] = sum_d dO * O, one warp per row.
template <typename T>
__global__ void __launch_bounds__(256) delta_kernel(const __grid_constant__ Params p, float* delta) {
  const int64_t nrow = (int64_t)p.B * p.H * p.Sq;
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  tc::pdl_wait();
  tc::pdl_trigger();
  if (row >= nrow) return;
  const int64_t i = row % p.Sq, bh = row / p.Sq;
  const T* o = row_of<T>((const void*)p.o, p.o_s, (int)(bh / p.H), (int)(bh % p.H), i);
  const float* o32 = p.o32 ? p.o32 + row * p.D : nullptr;
  const T* g = row_of<T>(p.d_o, p.do_s, (int)(bh / p.H), (int)(bh % p.H), i);
  float s = 0.f;
  for (int d = lane; d < p.D; d += 32) s = fmaf(o32 ? o32[d] : to_f32<T>(o[d]), to_f32<T>(g[d]), s);
  s = warp_sum(s);
  if (lane == 0) delta[row] = s;
}

// dtable[n][h] = sum over batch and query tiles of the partial sums, one warp per (n, h), a fixed order.
__global__ void __launch_bounds__(256) dtable_kernel(const float* __restrict__ part, float* __restrict__ dtable, int B,
                                                     int H, int nt, int nb) {
  const int lane = threadIdx.x & 31;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5);
  tc::pdl_wait();
  tc::pdl_trigger();
  if (w >= nb * H) return;
  const int n = w / H, h = w % H;
  float s = 0.f;
  for (int64_t i = lane; i < (int64_t)B * nt; i += 32)
    s += part[((i / nt * H + h) * nt + i % nt) * nb + n];
  s = warp_sum(s);
  if (lane == 0) dtable[n * H + h] = s;
}

__global__ void __launch_bounds__(256) zero_rows_kernel(uint8_t* o, int64_t s0, int64_t s1, int64_t s2, int H, int64_t S,
                                                        int64_t n, int row_bytes) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / row_bytes, bh = row / S;
    o[(bh / H) * s0 + (bh % H) * s1 + (row % S) * s2 + i % row_bytes] = 0;
  }
}

int zero_rows(void* t, const int64_t* s, int64_t B, int64_t H, int64_t S, int64_t D, int dtype, cudaStream_t st) {
  const int64_t es = (int64_t)dtype_size(dtype), n = B * H * S * D * es;
  if (!t || n == 0) return 0;
  {
    LaunchScope ls("bias_attn_zero", st);
    zero_rows_kernel<<<grid_for(n, 256, 16), 256, 0, st>>>((uint8_t*)t, s[0] * es, s[1] * es, s[2] * es, (int)H, S, n,
                                                          (int)(D * es));
  }
  return after_launch("bias_attn_zero");
}

int check(const b2_bias_attn_args* a, bool bwd) {
  const char* w = bwd ? "bias_attn_bwd" : "bias_attn_fwd";
  if (!a) return fail(B2_ERR_ARG, std::string(w) + ": null arguments");
  if (a->dtype != B2_F32 && a->dtype != B2_BF16 && a->dtype != B2_F16)
    return fail(B2_ERR_ARG, std::string(w) + ": dtype must be F32, BF16 or F16");
  if (a->B < 0 || a->H < 0 || a->Hk < 0 || a->Sq < 0 || a->Sk < 0)
    return fail(B2_ERR_ARG, std::string(w) + ": negative size");
  if (a->D < 1 || a->D > 128) return fail(B2_ERR_ARG, std::string(w) + ": head dim must be 1..128");
  if (a->H > 0 && (a->Hk < 1 || a->H % a->Hk))
    return fail(B2_ERR_ARG, std::string(w) + ": the query heads must be a multiple of the key/value heads");
  if (a->B * a->H > 65535) return fail(B2_ERR_ARG, std::string(w) + ": batch * heads must be at most 65535");
  if (a->Sq >= (1ll << 29) || a->Sk >= (1ll << 29) || a->q_offset >= (1ll << 29) || a->q_offset <= -(1ll << 29))
    return fail(B2_ERR_ARG, std::string(w) + ": lengths and q_offset must be below 2^29");
  if (!bucket_args_ok(a->num_buckets, a->max_distance, a->bidirectional))
    return fail(B2_ERR_ARG, std::string(w) + ": num_buckets must be 2..128 (two-sided: even, 4..128) and max_distance "
                                             "above half a side's buckets and at most 1024");
  if (a->B == 0 || a->H == 0 || a->Sq == 0) return 0;
  if ((uintptr_t)a->o32 & 15) return fail(B2_ERR_ARG, std::string(w) + ": o32 must be 16-byte aligned");
  if (!a->q || (!a->o && !(bwd && a->o32)) || !a->table || (a->Sk > 0 && (!a->k || !a->v)))
    return fail(B2_ERR_ARG, std::string(w) + ": null tensor");
  if (bwd && (!a->d_o || !a->lse)) return fail(B2_ERR_ARG, std::string(w) + ": dO and lse are required");
  return 0;
}

struct Plan {
  bool tc = false, rows = false;
  int nsplit = 1;
  int ntq = 0;               // query tiles of the bias-gradient partial sums
  int sq_pad = 0;            // tensor-core backward: rows of (lse, delta) per head
  uint64_t part_o = 0, part_ml = 0, delta = 0, dtab = 0, norms = 0, bytes = 0;  // offsets into the workspace
};

uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

// Key splits of the forward: the waves of blocks times the key tiles a block walks plus 1.6 us of set-up,
// and for the join its bytes (each split's fp32 output written and read) at the memory's rate, where a tile takes about
// 0.4 us on the tensor cores and 3 us on the FMA pipe, and a launch. At least two tiles a split. Measured, 16 heads x 4096 x
// 4096: 2 splits save a sixth of the walk (3.5 waves) and their join takes 47 us of it back.
int pick_splits(int64_t blocks, int64_t tk, int64_t out_elems, double tile_us) {
  const int64_t sms = 2 * (device_info().sm_count > 0 ? device_info().sm_count : 148);  // two blocks to an SM
  int best = 1;
  double best_cost = 1e30;
  for (int64_t ns = 1; ns <= std::max<int64_t>(1, std::min<int64_t>(tk / 2, 64)); ++ns) {
    const double join = ns > 1 ? (3.0 + (double)ns * out_elems * 8.0 / 3e6) / tile_us : 0.0;
    const double cost = (double)((blocks * ns + sms - 1) / sms) * ((tk + ns - 1) / ns + 1.6 / tile_us) + join;
    if (cost < best_cost) best_cost = cost, best = (int)ns;
  }
  return best;
}

Plan make_plan(const b2_bias_attn_args* a, bool bwd) {
  Plan pl;
  const int64_t rows = a->B * a->H * a->Sq;
  pl.tc = bwd ? tc_bwd_eligible(a) : tc_fwd_eligible(a);
  const int tile = pl.tc ? kTcTile : kSimtTile;
  const int64_t walk = pl.tc ? kTcTile : kSimtWalk;
  const int64_t tq = (a->Sq + tile - 1) / tile, tk = (a->Sk + walk - 1) / walk;
  if (!bwd && rows_eligible(a)) {
    // Few query rows. An SM holds `res` blocks at a time and needs two thirds of them to keep the memory busy, so a last,
    // partly filled round counts as that many; a block costs its keys and about 75 keys' worth of set-up, the join 64 + 4 ns.
    // 8 x 16 heads over 8192 keys: 50.2, 52.2, 48.0, 49.8 and 51.8 us with 6, 7, 11, 13 and 24 splits.
    pl.rows = true;
    const int64_t groups = (a->Sq * (a->H / a->Hk) + 7) / 8;
    const int64_t blocks = a->B * a->Hk * groups, sms = device_info().sm_count > 0 ? device_info().sm_count : 148;
    const int64_t res = rows_blocks_per_sm(a), least = (2 * res + 2) / 3;
    int64_t best = INT64_MAX;
    for (int64_t ns = 1; ns <= std::max<int64_t>(1, std::min<int64_t>(a->Sk / 64, 128)); ++ns) {
      const int64_t full = blocks * ns / (sms * res), rest = (blocks * ns - full * sms * res + sms - 1) / sms;
      const int64_t cost = (full * res + (rest ? std::max(rest, least) : 0)) * ((a->Sk + ns - 1) / ns + 75) + (ns > 1 ? 64 + 4 * ns : 0);
      if (cost < best) best = cost, pl.nsplit = (int)ns;
    }
  } else if (!bwd) {
    pl.nsplit = pick_splits(tq * a->B * a->H, tk, rows * a->D, pl.tc ? 0.4 : 3.0);
  } else {
    pl.ntq = (int)tq;
    pl.delta = 0;
    pl.sq_pad = (int)((a->Sq + kTcPad - 1) / kTcPad * kTcPad);
    pl.dtab = pl.tc ? (uint64_t)(a->B * a->H) * pl.sq_pad * 8 : up16((uint64_t)rows * 4);
    pl.norms = pl.dtab + (a->dtable ? up16((uint64_t)(a->B * a->H * tq) * a->num_buckets * 4) : 0);
    pl.bytes = pl.norms + (pl.tc && a->dtype == B2_F16 ? up16((uint64_t)(a->B * a->Hk) * 8) : 0);
  }
  if (pl.nsplit > 1) {
    pl.part_o = 0;
    pl.part_ml = up16((uint64_t)pl.nsplit * rows * a->D * 4);
    pl.bytes = pl.part_ml + up16((uint64_t)pl.nsplit * rows * 8);
  }
  return pl;
}

Params make_params(const b2_bias_attn_args* a) {
  Params p{};
  p.q = a->q, p.k = a->k, p.v = a->v, p.o = a->o, p.o32 = a->o32, p.lse = a->lse, p.table = a->table, p.mask = a->key_mask;
  p.d_o = a->d_o, p.dq = a->dq, p.dk = a->dk, p.dv = a->dv;
  for (int i = 0; i < 3; ++i) {
    p.q_s[i] = a->q_s[i], p.k_s[i] = a->k_s[i], p.v_s[i] = a->v_s[i], p.o_s[i] = a->o_s[i];
    p.do_s[i] = a->do_s[i], p.dq_s[i] = a->dq_s[i], p.dk_s[i] = a->dk_s[i], p.dv_s[i] = a->dv_s[i];
  }
  p.mask_sb = a->mask_sb;
  p.B = (int)a->B, p.H = (int)a->H, p.Hk = (int)a->Hk, p.Sq = (int)a->Sq, p.Sk = (int)a->Sk, p.D = (int)a->D;
  p.q_off = (int)a->q_offset;
  p.R = a->max_distance;
  p.nb = a->num_buckets;
  p.bidir = a->bidirectional ? 1 : 0, p.causal = a->causal ? 1 : 0;
  p.nsplit = 1;
  {
    // a function of the two numbers alone, remembered per thread: its logarithms cost more than a launch
    thread_local int nb = 0, dist = 0, n = 0;
    thread_local uint16_t thr[B2_BIAS_MAX_BUCKETS];
    const int side = p.bidir ? p.nb / 2 : p.nb;
    if (nb != side || dist != p.R) n = thresholds(side, p.R, thr), nb = side, dist = p.R;
    p.nthr = n;
    std::copy(thr, thr + n, p.thr);
  }
  p.scale = a->scale;
  p.err = device_error_ptr();
  return p;
}

template <template <typename> class F, typename... A>
int by_dtype(int dt, A&&... args) {
  switch (dt) {
    case B2_F32: return F<float>::run(args...);
    case B2_BF16: return F<__nv_bfloat16>::run(args...);
    default: return F<__half>::run(args...);
  }
}

template <typename T>
struct Combine {
  static int run(const Params& p, cudaStream_t st) {
    return launch_pdl("bias_attn_combine", combine_kernel<T>, dim3((unsigned)(p.B * p.H * (int64_t)p.Sq)), dim3(128), 0, st, p);
  }
};
template <typename T>
struct Delta {
  static int run(const Params& p, float* delta, cudaStream_t st) {
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    return launch_pdl("bias_attn_delta", delta_kernel<T>, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, st, p, delta);
  }
};

int need_workspace(const b2_bias_attn_args* a, const Plan& pl, const char* w) {
  if (pl.bytes && (!a->workspace || ((uintptr_t)a->workspace & 15)))
    return fail(B2_ERR_ARG, std::string(w) + ": a 16-byte aligned workspace of b2_bias_attn_workspace_bytes() is required");
  return 0;
}

}  // namespace
}  // namespace bias_attn
}  // namespace b2

extern "C" int b2_bias_bucket(int64_t rel, int32_t num_buckets, int32_t max_distance, int32_t bidirectional) {
  using namespace b2::bias_attn;
  if (!bucket_args_ok(num_buckets, max_distance, bidirectional)) return -1;
  uint16_t thr[B2_BIAS_MAX_BUCKETS];
  const int side = bidirectional ? num_buckets / 2 : num_buckets;
  const int n = thresholds(side, max_distance, thr);
  const int64_t d = bidirectional ? (rel < 0 ? -rel : rel) : (rel < 0 ? -rel : 0);
  int c = 0;
  for (int i = 0; i < n; ++i) c += d >= (int64_t)thr[i];
  return c + (bidirectional && rel > 0 ? side : 0);
}

extern "C" uint64_t b2_bias_attn_workspace_bytes(const b2_bias_attn_args* a, int32_t backward) {
  using namespace b2::bias_attn;
  if (!a || a->B <= 0 || a->H <= 0 || a->Sq <= 0 || a->Sk <= 0) return 0;
  if (check(a, backward != 0)) return 0;
  b2::ensure_init();
  return make_plan(a, backward != 0).bytes;
}

extern "C" int b2_bias_attn_fwd(const b2_bias_attn_args* a, b2_stream_t stream) {
  using namespace b2;
  using namespace b2::bias_attn;
  if (int rc = check(a, false)) return rc;
  if (int rc = ensure_init()) return rc;
  if (a->B == 0 || a->H == 0 || a->Sq == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  const Plan pl = make_plan(a, false);
  if (int rc = need_workspace(a, pl, "bias_attn_fwd")) return rc;
  Params p = make_params(a);
  p.nsplit = pl.nsplit;
  p.part_o = (float*)((char*)a->workspace + pl.part_o);
  p.part_ml = (float2*)((char*)a->workspace + pl.part_ml);
  if (int rc = pl.rows ? rows_fwd(p, a->dtype, st) : pl.tc ? tc_fwd(p, a->dtype == B2_BF16, st) : simt_fwd(p, a->dtype, st))
    return rc;
  return p.nsplit > 1 ? by_dtype<Combine>(a->dtype, p, st) : 0;
}

extern "C" int b2_bias_attn_bwd(const b2_bias_attn_args* a, b2_stream_t stream) {
  using namespace b2;
  using namespace b2::bias_attn;
  if (int rc = check(a, true)) return rc;
  if (int rc = ensure_init()) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (a->B == 0 || a->H == 0 || a->Sq == 0 || a->Sk == 0) {
    // no pairs: whatever exists of the gradients is zero
    if (a->H > 0) {
      if (int rc = zero_rows(a->dq, a->dq_s, a->B, a->H, a->Sq, a->D, a->dtype, st)) return rc;
      if (int rc = zero_rows(a->dk, a->dk_s, a->B, a->Hk, a->Sk, a->D, a->dtype, st)) return rc;
      if (int rc = zero_rows(a->dv, a->dv_s, a->B, a->Hk, a->Sk, a->D, a->dtype, st)) return rc;
      if (a->dtable)
        return check_cuda(cudaMemsetAsync(a->dtable, 0, (size_t)a->num_buckets * a->H * 4, st), "bias_attn_bwd memset");
    }
    return 0;
  }
  const Plan pl = make_plan(a, true);
  if (int rc = need_workspace(a, pl, "bias_attn_bwd")) return rc;
  Params p = make_params(a);
  float* delta = (float*)((char*)a->workspace + pl.delta);
  p.delta = delta;
  p.dtab = a->dtable ? (float*)((char*)a->workspace + pl.dtab) : nullptr;
  if (pl.tc) {
    if (a->dtype == B2_F16) {
      p.norms = (uint32_t*)((char*)a->workspace + pl.norms);
      if (int rc = check_cuda(cudaMemsetAsync(p.norms, 0, (size_t)(a->B * a->Hk) * 8, st), "bias_attn_bwd memset")) return rc;
    }
    if (int rc = tc_bwd(p, a->dtype == B2_BF16, (float2*)delta, pl.sq_pad, st)) return rc;
  } else {
    if (int rc = by_dtype<Delta>(a->dtype, p, delta, st)) return rc;
    if (int rc = simt_bwd(p, a->dtype, st)) return rc;
  }
  if (a->dtable) {
    return launch_pdl("bias_attn_dtable", dtable_kernel, dim3((unsigned)((p.nb * p.H + 7) / 8)), dim3(256), 0, st,
                      (const float*)p.dtab, a->dtable, p.B, p.H, pl.ntq, p.nb);
  }
  return 0;
}
