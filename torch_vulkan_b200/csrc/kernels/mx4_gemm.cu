// Linear layers over a frozen MXFP4 weight W [N][K] on the tensor cores of sm_100a, the LoRA term in the same product:
//   forward  out[M][N] = A W^T + bias + h[M][r] b[N][r]^T     A an MXFP4 matrix [M][K]
//   dX       out[M][K] = dY[M][N] W + h[M][r] a[r][K]         dY bf16, W expanded to bf16 (exact) by a kernel before
//
// Forward: tcgen05.mma.kind::mxf4.block_scale multiplies E2M1 codes and applies the two E8M0 scales of every 32 products
// itself, with fp32 accumulation in TMEM; a K block of 256 columns is 128 bytes a row. The scale of row r of a 128-row block
// stands in TMEM at lane r % 32 (of all four lane quarters), column r / 32, one byte per block of 32 columns, which is the
// order the scale array is stored in: four warps copy each stage's 512-byte pieces with one 16-byte load per lane and
// tcgen05.st. (tcgen05.cp 32x128b.warpx4 does the same from the MMA thread, but its copies and the MMAs do not overlap:
// 0.49 us a stage for the six of a 256 x 256 pair tile next to 0.52 us of MMAs, 0.75 us together.) dX: W's scales run along its output, not along the
// reduction, so the block-scaled MMA cannot apply them: kind::f16 with W as the N-major operand. The LoRA term is one more
// K block of bf16 operands, zero-filled past r, into the same accumulator: one rounding for the sum.
//
// Persistent CTAs, or CTA pairs (CG = 2: each CTA stages its own 128 rows of A and half of the W tile, the leader issues
// M = 256 MMAs for both; W's scales are needed whole in each). warp 0: TMA producer. warp 1: MMAs. warps 10..13: scales.
// warps 2..9: epilogue, which takes the whole tile into registers as bf16 before it stores anything, so that the next
// tile's MMAs wait for a few hundred cycles only.
#include "common.cuh"
#include "tc_ptx.cuh"

namespace b2 {

bool make_tmap(CUtensorMap* m, CUtensorMapDataType dt, int rank, const void* base, const uint64_t* dims,
               const uint64_t* strides_bytes, const uint32_t* box, CUtensorMapSwizzle sw);  // gemm_tc.cu

namespace {

struct P4 {
  const __nv_bfloat16* bias;
  __nv_bfloat16* out;
  int64_t out_ld;
  int M, NO;          // rows and columns of the output
  int KR;             // reduction: columns padded to 32 (forward), N (dX)
  int tiles_m, tiles_n;
  int lora_r;
  int vec_out;        // rows of out are whole 16-byte groups
  int* err;
};

// MS: 128-row sub-tiles of A per CTA that share the stage's W tile.
template <int BN, int CG, int MS, bool DX>
struct Cfg4 {
  static constexpr int BMC = 128 * MS;                 // rows of a tile in this CTA
  static constexpr int BM = BMC * CG;                  // rows of a tile
  static constexpr int BK = DX ? 64 : 256;             // reduction per K block: 128 bytes a row
  static constexpr int BC = BN / CG;                   // rows of W (dX: columns) that this CTA stages
  static constexpr int A_BYTES = BMC * 128, B_BYTES = BC * 128;
  static constexpr int SA_BYTES = DX ? 0 : 1024, SB_BYTES = DX ? 0 : 1024 * (BN / 128);
  static constexpr int TX = A_BYTES + B_BYTES;
  static constexpr int STAGE = TX + SA_BYTES + SB_BYTES;
  static constexpr int NS = MS == 2 ? 4 : (BN / CG == 64 ? 6 : 5);
  static constexpr int NACC = MS == 2 ? 1 : 256 / BN;  // accumulators in TMEM, MS * BN columns each
  static constexpr int SFC = DX ? 0 : 8 + BN / 16;     // TMEM columns of a stage's scales (A: 2 x 4, W: 2 x BN / 32)
  static constexpr uint32_t T_SF = 256, TMEM_COLS = 512;
  static_assert((DX || MS == 1) && MS * BN <= 512 && (DX || T_SF + NS * SFC <= 512), "TMEM columns");
  static constexpr int OFF_STG = NS * STAGE;           // 8 warps x a 4 KB box
  static constexpr int OFF_BIAS = OFF_STG + 8 * 4096;  // 2 x BN floats
  static constexpr int OFF_BAR = OFF_BIAS + (DX ? 0 : 2 * BN * 4);
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory");
  static_assert(STAGE % 1024 == 0, "swizzled tiles start on 1024-byte boundaries");
  static constexpr int THREADS = DX ? 320 : 448;
};

// Instruction descriptor of kind::mxf4 (PTX ISA, block-scaled kinds): [4,6) scale id of B | [7,10) A format, 1 = E2M1 |
// [10,12) B format | [17,23) N >> 3 | [23] 1 = UE8M0 scales | [24,29) M >> 4 | [29,31) scale id of A. The scale id is the
// byte of a scale column's words at which the two scales of this MMA's 64 columns start (0 or 2).
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int sf) {
  return ((uint32_t)sf << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 4) << 24) |
         ((uint32_t)sf << 29);
}

template <int CG>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t acc) {
  if (CG == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(sfa), "r"(sfb)
        : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_bf16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if (CG == 2) tc::mma_f16_ss_pair(d, a, b, idesc, acc);
  else tc::mma_f16_ss(d, a, b, idesc, acc);
}

template <int BN, int CG, int MS, bool DX>
__global__ void __launch_bounds__(DX ? 320 : 448, 1)
    mx4_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSW,
                    const __grid_constant__ CUtensorMap tmH, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ P4 p) {
  using C = Cfg4<BN, CG, MS, DX>;
  constexpr int NS = C::NS, NACC = C::NACC;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);  // [NS] (pairs: the leader's, for both CTAs' bytes)
  uint64_t* empty = full + NS;                                      // [NS]
  uint64_t* acc_full = empty + NS;                                  // [2]
  uint64_t* acc_empty = acc_full + 2;                               // [2] one arrival per epilogue warp (of both CTAs)
  uint64_t* sfull = acc_empty + 2;                                  // [NS] this CTA's scales of a stage landed
  uint64_t* sready = sfull + NS;                                    // [NS] and are in TMEM (pairs: in both CTAs' TMEM)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(sready + NS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(sready + NS + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? tc::cluster_ctarank() : 0u;
  auto leader_bar = [&](uint64_t* bar) -> uint32_t {
    return CG == 2 ? tc::mapa_shared(tc::smem_u32(bar), 0u) : tc::smem_u32(bar);
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      tc::mbar_init(&full[i], 1), tc::mbar_init(&empty[i], 1);
      tc::mbar_init(&sfull[i], 1), tc::mbar_init(&sready[i], 4 * CG);
    }
    for (int i = 0; i < 2; ++i) tc::mbar_init(&acc_full[i], 1), tc::mbar_init(&acc_empty[i], 8 * CG);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  if (CG == 2) tc::cluster_sync();  // both CTAs' barriers are ready before any arrival from the other
  tc::pdl_wait();
  if (warp == 1) {
    if (CG == 2) {
      tc::tmem_alloc_pair(tmem_slot, C::TMEM_COLS);
      tc::tmem_relinquish_pair();
    } else {
      tc::tmem_alloc(tmem_slot, C::TMEM_COLS);
      tc::tmem_relinquish();
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tbase = *tmem_slot;
  tc::pdl_trigger();

  const int tiles = p.tiles_m * p.tiles_n;
  const int nkm = (p.KR + C::BK - 1) / C::BK;  // K blocks of the main product
  const int nk = nkm + (p.lora_r ? 1 : 0);
  const int unit = (int)blockIdx.x / CG, units = (int)gridDim.x / CG;
  // consecutive units take consecutive row tiles of one column of tiles, so they share W in L2
  auto tile_m = [&](int t) { return t % p.tiles_m * C::BM + (int)rank * C::BMC; };  // this CTA's first row
  auto tile_n = [&](int t) { return t / p.tiles_m * BN; };

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- producer ----------------
      int it = 0;
      int issued[NS] = {};
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units) {
        const int m0 = tile_m(t), n0 = tile_n(t), nb0 = n0 + (int)rank * C::BC;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % NS;
          if (!tc::mbar_wait(&empty[s], (uint32_t)((it / NS) & 1) ^ 1, p.err) || *abort_flag) { ok = false; break; }
          uint8_t* st = smem + s * C::STAGE;
          uint8_t* sb = st + C::A_BYTES;
          uint8_t* sc = sb + C::B_BYTES;
          const bool lora = kb == nkm;
          if (rank == 0) tc::mbar_arrive_expect_tx(&full[s], C::TX * CG);
          auto load = [&](void* dst, const CUtensorMap* m, int x, int y) {
            if (CG == 2) tc::tma_load_2d_pair(dst, m, leader_bar(&full[s]), x, y);
            else tc::tma_load_2d(dst, m, &full[s], x, y);
          };
          if (DX) {
            load(st, lora ? &tmH : &tmA, lora ? 0 : kb * 64, m0);
            for (int c = 0; c < C::BC / 64; ++c)  // 64 rows x 64 columns per box
              load(sb + c * 8192, lora ? &tmB : &tmW, nb0 + c * 64, lora ? 0 : kb * 64);
          } else if (lora) {
            tc::mbar_arrive(&sfull[s]);  // no scales
            load(st, &tmH, 0, m0);
            load(sb, &tmB, 0, nb0);
          } else {
            tc::mbar_arrive_expect_tx(&sfull[s], C::SA_BYTES + C::SB_BYTES);
            tc::tma_load_2d(sc, &tmSA, &sfull[s], kb * 256, m0 / 128);
            tc::tma_load_2d(sc + 1024, &tmSW, &sfull[s], kb * 256, n0 / 128);
            load(st, &tmA, kb * 128, m0);
            load(sb, &tmW, kb * 128, nb0);
          }
          issued[s]++;
        }
      }
      if (ok && CG == 2) {
        // the leader's last commits arrive on this CTA's barriers: wait for them before the CTA can leave
        for (int s = 0; s < NS; ++s)
          if (issued[s]) tc::mbar_wait(&empty[s], (uint32_t)((issued[s] - 1) & 1), p.err);
      }
      if (!ok) {
        *abort_flag = 1;
        for (int s = 0; s < NS; ++s)
          if (issued[s]) {
            if (rank == 0) tc::mbar_wait(&full[s], (uint32_t)((issued[s] - 1) & 1), nullptr);
            if (!DX) tc::mbar_wait(&sfull[s], (uint32_t)((issued[s] - 1) & 1), nullptr);
          }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // ---------------- MMA issuer (pairs: the leader) ----------------
      constexpr uint32_t ID0 = idesc_mxf4(128 * CG, BN, 0), ID2 = idesc_mxf4(128 * CG, BN, 2);
      constexpr uint32_t IDF = tc::idesc_f16(128 * CG, BN, true, false, DX);
      int it = 0, ti = 0;
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units, ++ti) {
        const int a = ti % NACC;
        if (!tc::mbar_wait(&acc_empty[a], (uint32_t)((ti / NACC) & 1) ^ 1, p.err)) { ok = false; break; }
        tc::tc_fence_after();
        const uint32_t acc = tbase + a * BN;
        for (int kb = 0; kb < nk; ++kb, ++it) {
          const int s = it % NS;
          if (!tc::mbar_wait(&full[s], (uint32_t)((it / NS) & 1), p.err) ||
              (!DX && !tc::mbar_wait(&sready[s], (uint32_t)((it / NS) & 1), p.err)) || *abort_flag) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t st = tc::smem_u32(smem + s * C::STAGE);
          const tc::SDesc ad = tc::sdesc_parts(st, 16, 1024);
          const bool lora = kb == nkm;
          if (DX || lora) {
            const tc::SDesc bd = tc::sdesc_parts(st + C::A_BYTES, DX ? 8192 : 16, 1024);
            const int steps = min(4, ((lora ? p.lora_r : p.KR - kb * 64) + 15) / 16);
            for (int k = 0; k < steps; ++k)
#pragma unroll
              for (int m = 0; m < MS; ++m)
                mma_bf16<CG>(acc + m * BN, tc::sdesc_at(ad, m * 16384 + k * 32), tc::sdesc_at(bd, DX ? k * 2048 : k * 32), IDF,
                             (kb > 0 || k > 0) ? 1u : 0u);
          } else {
            const tc::SDesc bd = tc::sdesc_parts(st + C::A_BYTES, 16, 1024);
            const uint32_t sfa = tbase + C::T_SF + s * C::SFC, sfb = sfa + 8;
            const int steps = min(4, (p.KR - kb * C::BK + 63) / 64);
            for (int k = 0; k < steps; ++k)
              mma_mxf4<CG>(acc, tc::sdesc_at(ad, k * 32), tc::sdesc_at(bd, k * 32), (k & 1) ? ID2 : ID0, sfa + 4 * (k >> 1),
                           sfb + (BN / 32) * (k >> 1), (kb > 0 || k > 0) ? 1u : 0u);
          }
          if (CG == 2) tc::mma_commit_pair(&empty[s], (uint16_t)3);
          else tc::mma_commit(&empty[s]);
        }
        if (ok) {
          if (CG == 2) tc::mma_commit_pair(&acc_full[a], (uint16_t)3);
          else tc::mma_commit(&acc_full[a]);
        }
      }
      if (!ok) *abort_flag = 1;
    }
  } else if (!DX && warp >= 10) {
    // ---------------- scales: warp = one lane quarter of TMEM ----------------
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    int it = 0;
    bool ok = true;
    for (int t = unit; t < tiles && ok; t += units)
      for (int kb = 0; kb < nk; ++kb, ++it) {
        const int s = it % NS;
        // its slot in TMEM is free: the loads waited for the MMAs that read the slot before
        if (!tc::mbar_wait(&sfull[s], (uint32_t)((it / NS) & 1), p.err) || *abort_flag) { ok = false; break; }
        if (kb < nkm) {
          const uint8_t* sc = smem + s * C::STAGE + C::A_BYTES + C::B_BYTES + lane * 16;
          uint32_t va[8], vb[BN / 16];
#pragma unroll
          for (int c = 0; c < 2; ++c) {  // 128-column pieces
            *reinterpret_cast<uint4*>(va + 4 * c) = *reinterpret_cast<const uint4*>(sc + 512 * c);
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)
              *reinterpret_cast<uint4*>(vb + (BN / 32) * c + 4 * j) = *reinterpret_cast<const uint4*>(sc + 1024 * (1 + j) + 512 * c);
          }
          __syncwarp();
          const uint32_t sf = tbase + C::T_SF + s * C::SFC + lane_off;
          tc::tmem_st8(sf, va);
          if (BN == 256) tc::tmem_st16(sf + 8, vb);
          else tc::tmem_st8(sf + 8, vb);
          tc::tmem_wait_st();
          tc::tc_fence_before();
        }
        __syncwarp();
        if (lane == 0) {
          if (CG == 2) tc::mbar_arrive_cluster(leader_bar(&sready[s]));
          else tc::mbar_arrive(&sready[s]);
        }
      }
    if (!ok) *abort_flag = 1;
  } else {
    // ---------------- epilogue: warp = 32 rows (TMEM lane quarter) x half of the columns ----------------
    const int half = (warp - 2) >> 2, quarter = warp & 3;
    const uint32_t lane_off = (uint32_t)(quarter * 32) << 16;
    const int ew = (int)threadIdx.x - 64;
    uint8_t* stg = smem + C::OFF_STG + (warp - 2) * 4096;
    float* bias_s = reinterpret_cast<float*>(smem + C::OFF_BIAS);
    constexpr int BOX = BN / 64;  // 32-column boxes of this warp
    int ti = 0;
    for (int t = unit; t < tiles; t += units, ++ti) {
      const int m0 = tile_m(t), n0 = tile_n(t), a = ti % NACC;
      float* bs = bias_s + (ti & 1) * BN;
      if (!DX) {
        if (ew < BN) bs[ew] = (p.bias && n0 + ew < p.NO) ? __bfloat162float(p.bias[n0 + ew]) : 0.f;
        tc::named_bar_sync(1, 256);
      }
      // after a wait that ran out, the remaining tiles are walked without waiting or storing: every warp still meets
      // the others at the named barrier
      const bool ok = !*abort_flag && tc::mbar_wait(&acc_full[a], (uint32_t)((ti / NACC) & 1), p.err);
      if (!ok) *abort_flag = 1;
      tc::tc_fence_after();
#pragma unroll 1
      for (int ms = 0; ms < MS; ++ms) {
        // half a row of the sub-tile into registers as bf16 pairs, so that the accumulator is free before the last
        // sub-tile is stored
        uint32_t w[BOX][16];
        __syncwarp();
#pragma unroll
        for (int c = 0; c < BOX; ++c) {
          uint32_t v[32];
          tc::tmem_ld32(tbase + (a * MS + ms) * BN + half * (BN / 2) + c * 32 + lane_off, v);
          tc::tmem_wait_ld();
          tc::reg_fence32(v);
          const float4* bc = reinterpret_cast<const float4*>(bs + half * (BN / 2) + c * 32);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float2 lo = make_float2(__uint_as_float(v[4 * e]), __uint_as_float(v[4 * e + 1]));
            float2 hi = make_float2(__uint_as_float(v[4 * e + 2]), __uint_as_float(v[4 * e + 3]));
            if (!DX) {
              const float4 bq = bc[e];
              lo = __fadd2_rn(lo, make_float2(bq.x, bq.y)), hi = __fadd2_rn(hi, make_float2(bq.z, bq.w));
            }
            __nv_bfloat162 p0 = __floats2bfloat162_rn(lo.x, lo.y), p1 = __floats2bfloat162_rn(hi.x, hi.y);
            w[c][2 * e] = *reinterpret_cast<uint32_t*>(&p0), w[c][2 * e + 1] = *reinterpret_cast<uint32_t*>(&p1);
          }
        }
        if (ms == MS - 1) {
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 2) tc::mbar_arrive_cluster(leader_bar(&acc_empty[a]));
            else tc::mbar_arrive(&acc_empty[a]);
          }
        }
        if (!ok) continue;
        const int r0 = m0 + ms * 128 + quarter * 32;
#pragma unroll
        for (int c = 0; c < BOX; c += 2) {
          // 32 rows x 64 columns through a swizzled staging tile, then whole 128-byte lines per row. Plain stores:
          // nothing waits for them, where a tile store's staging buffer is held until it has been read
          const int col = n0 + half * (BN / 2) + c * 32;
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t* v = &w[c + (e >> 2)][4 * (e & 3)];
            *reinterpret_cast<uint4*>(stg + lane * 128 + ((e ^ (lane & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
          }
          __syncwarp();
          if (p.vec_out) {
            const int cc = col + (lane & 7) * 8;  // NO is a multiple of 8 here: an 8-column group is whole or absent
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = i * 4 + (lane >> 3);
              const uint4 v = *reinterpret_cast<const uint4*>(stg + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
              if (r0 + r < p.M && cc < p.NO) *reinterpret_cast<uint4*>(p.out + (int64_t)(r0 + r) * p.out_ld + cc) = v;
            }
          } else {
#pragma unroll 4
            for (int r = 0; r < 32; ++r) {
              if (r0 + r >= p.M) break;
              __nv_bfloat16* o = p.out + (int64_t)(r0 + r) * p.out_ld;
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const int e = lane + 32 * j;
                const __nv_bfloat16 v = *reinterpret_cast<const __nv_bfloat16*>(stg + r * 128 + (((e >> 3) ^ (r & 7)) << 4) + (e & 7) * 2);
                if (col + e < p.NO) o[col + e] = v;
              }
            }
          }
        }
      }
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (CG == 2) tc::cluster_sync();  // neither CTA leaves while the other may still arrive on its barriers
  if (warp == 1) {
    __syncwarp();
    tc::tc_fence_after();
    if (CG == 2) tc::tmem_dealloc_pair(tbase, C::TMEM_COLS);
    else tc::tmem_dealloc(tbase, C::TMEM_COLS);
  }
}

bool map2d(CUtensorMap* m, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t rows, uint64_t ld_bytes,
           uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle sw) {
  const uint64_t dims[2] = {inner, rows};
  const uint64_t strides[1] = {ld_bytes};
  const uint32_t box[2] = {box_inner, box_rows};
  return make_tmap(m, dt, 2, base, dims, strides, box, sw);
}

// Output dimensions, operands and leading dims of either direction.
struct Shape {
  int64_t NO, KR;
  const void* x;     // dX: bf16 dY rows
  int64_t x_ld;
  const void* w;     // dX: expanded weight
  int64_t w_ld;
};

template <int BN, int CG, int MS, bool DX>
int launch4(const b2_mx4_gemm_args* a, const Shape& sh, cudaStream_t st) {
  using C = Cfg4<BN, CG, MS, DX>;
  const char* name = DX ? "mx4_gemm_dx" : "mx4_gemm";
  auto kern = mx4_gemm_kernel<BN, CG, MS, DX>;
  if (int rc = allow_smem<mx4_gemm_kernel<BN, CG, MS, DX>>(C::SMEM, name)) return rc;
  P4 p{};
  p.bias = DX ? nullptr : (const __nv_bfloat16*)a->bias;
  p.out = (__nv_bfloat16*)a->out, p.out_ld = a->out_ld;
  p.M = (int)a->M, p.NO = (int)sh.NO, p.KR = (int)sh.KR;
  p.tiles_m = (int)((a->M + C::BM - 1) / C::BM), p.tiles_n = (int)((sh.NO + BN - 1) / BN);
  p.lora_r = a->lora_r;
  p.err = device_error_ptr();
  p.vec_out = a->out_ld % 8 == 0 && sh.NO % 8 == 0 && ((uintptr_t)a->out & 15) == 0;
  CUtensorMap ta, tw, tsa, tsw, th, tb;
  for (CUtensorMap* m : {&tsa, &tsw, &th, &tb}) memset(m, 0, sizeof(*m));
  const auto U8 = CU_TENSOR_MAP_DATA_TYPE_UINT8, BF = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, I32 = CU_TENSOR_MAP_DATA_TYPE_INT32;
  const auto S128 = CU_TENSOR_MAP_SWIZZLE_128B, S0 = CU_TENSOR_MAP_SWIZZLE_NONE;
  bool ok;
  if (DX) {
    ok = map2d(&ta, BF, sh.x, a->N, a->M, sh.x_ld * 2, 64, C::BMC, S128) && map2d(&tw, BF, sh.w, a->K, a->N, sh.w_ld * 2, 64, 64, S128);
  } else {
    const int64_t cb = b2_mx4_code_bytes(a->K), nkb = (a->K + 127) / 128;
    ok = map2d(&ta, U8, a->x_codes, cb, a->M, cb, 128, 128, S128) && map2d(&tw, U8, a->w_codes, cb, a->N, cb, 128, C::BC, S128) &&
         map2d(&tsa, I32, a->x_scales, nkb * 128, (a->M + 127) / 128, nkb * 512, 256, 1, S0) &&
         map2d(&tsw, I32, a->w_scales, nkb * 128, (a->N + 127) / 128, nkb * 512, 256, BN / 128, S0);
  }
  if (a->lora_r) {
    ok = ok && map2d(&th, BF, a->lora_h, a->lora_r, a->M, a->lora_h_ld * 2, 64, C::BMC, S128);
    ok = ok && (DX ? map2d(&tb, BF, a->lora_b, a->K, a->lora_r, a->lora_b_ld * 2, 64, 64, S128)
                   : map2d(&tb, BF, a->lora_b, a->lora_r, a->N, a->lora_b_ld * 2, 64, C::BC, S128));
  }
  if (!ok) return fail(B2_ERR_ARG, std::string(name) + ": tensor map rejected");
  const int units = std::min(p.tiles_m * p.tiles_n, device_info().sm_count / CG);
  if (CG == 1) return launch_pdl(name, kern, dim3(units), dim3(C::THREADS), C::SMEM, st, ta, tw, tsa, tsw, th, tb, p);
  // clusters of two; programmatic dependent launch as for single CTAs (outside stream capture)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(units * CG);
  cfg.blockDim = dim3(C::THREADS);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  if (cudaStreamIsCapturing(st, &cs) != cudaSuccess) {
    (void)cudaGetLastError();
    cs = cudaStreamCaptureStatusActive;
  }
  cfg.attrs = at;
  cfg.numAttrs = (pdl_enabled() && cs == cudaStreamCaptureStatusNone) ? 2 : 1;
  cudaError_t e;
  {
    LaunchScope ls(name, st);
    e = cudaLaunchKernelEx(&cfg, kern, ta, tw, tsa, tsw, th, tb, p);
  }
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail_cuda(e, name);
  }
  return after_launch(name);
}

// The tile whose waves cost least. A K block costs a CTA the longer of its MMAs and its operand loads: L2 feeds an SM
// about 75 KB per microsecond when all of them load (measured: 70 to 87), 256 columns of a 128-row MMA take 0.27 us for 64
// bf16 products and 0.52 us for 256 4-bit ones (as measured, the latter with the scales in place); each tile adds about
// 1.5 us of draining, and a pair launch about 1.2 us of cluster set-up. Measured: dX of 4096 x 8192 -> 2048 takes 129 us
// with 256 x 256 pair tiles (two waves) and 90 us with 512 x 256 ones (one wave); the forward of 1024 x 2048 -> 2048 takes
// 9.6 us with 256 x 128 pair tiles and 8.5 us with 128 x 128 ones.
struct Tile {
  int bn, cg, ms;
};
Tile pick_tile(int64_t M, int64_t NO, int64_t KR, bool dx) {
  static constexpr Tile cand[] = {{128, 1, 1}, {128, 2, 1}, {256, 2, 1}, {256, 2, 2}};
  Tile best = cand[0];
  double best_t = 1e30;
  const int64_t sms = device_info().sm_count;
  for (const Tile& c : cand) {
    if (c.ms == 2 && !dx) continue;
    const int64_t bm = 128 * c.ms * c.cg;
    const int64_t tiles = (M + bm - 1) / bm * ((NO + c.bn - 1) / c.bn);
    const int64_t waves = (tiles + sms / c.cg - 1) / (sms / c.cg);
    const double kb = (double)((KR + (dx ? 63 : 255)) / (dx ? 64 : 256));
    const double kbytes = 16.0 * c.ms + c.bn / c.cg / 8.0 + (dx ? 0.0 : 1.0 + c.bn / 128.0);
    const double mma = (dx ? 0.27 : 0.52) * c.ms * c.bn / 256;
    const double t = waves * (kb * std::max(mma, kbytes / 75.0) + 1.5 * c.ms * c.bn / 256 + 0.5) + (c.cg == 2 ? 1.2 : 0.0);
    if (t < best_t) best_t = t, best = c;
  }
  return best;
}

template <bool DX>
int launch_best(const b2_mx4_gemm_args* a, const Shape& sh, cudaStream_t st) {
  const Tile t = pick_tile(a->M, sh.NO, sh.KR, DX);
  if constexpr (DX)
    if (t.ms == 2) return launch4<256, 2, 2, true>(a, sh, st);
  if (t.bn == 256) return launch4<256, 2, 1, DX>(a, sh, st);
  return t.cg == 2 ? launch4<128, 2, 1, DX>(a, sh, st) : launch4<128, 1, 1, DX>(a, sh, st);
}

}  // namespace

// Sizes that the kernels' 32-bit tile arithmetic takes.
bool mx4_gemm_tc_eligible(const b2_mx4_gemm_args* a) {
  const int64_t lim = 1ll << 30;
  return device_info().tcgen05 && a->M < lim && a->N < lim && a->K < lim &&
         (a->M + 127) / 128 * ((std::max(a->N, a->K) + 127) / 128) < lim;
}

int mx4_gemm_fwd(const b2_mx4_gemm_args* a, cudaStream_t st) {
  return launch_best<false>(a, Shape{a->N, b2_mx4_code_bytes(a->K) * 2, nullptr, 0, nullptr, 0}, st);
}

// x: dY rows with a stride that is a multiple of 8 elements, 16-byte aligned; w: the expanded weight [N][w_ld]
int mx4_gemm_dx(const b2_mx4_gemm_args* a, const void* x, int64_t x_ld, const void* w, int64_t w_ld, cudaStream_t st) {
  return launch_best<true>(a, Shape{a->K, a->N, x, x_ld, w, w_ld}, st);
}

}  // namespace b2
