// MXFP4 (OCP microscaling): quantisation of a matrix to E2M1 codes with one power-of-two scale per 32 columns, and
// reading it back.
//
// A block's scale is 2^(floor(log2(amax)) - 2): with the fp32 exponent field e of amax that is the E8M0 code
// max(e - 2, 0), and multiplying by 2^(127 - code) divides exactly. The E2M1 rounding (nearest, ties to even,
// saturating) is the cvt.rn.satfinite.e2m1x2 instruction; reading back is one exact product per element.
#include "mx4.cuh"
#include "tc_ptx.cuh"

#include <type_traits>

namespace b2 {
namespace {

using namespace mx4;

// Eight consecutive elements at p as floats; `n` (< 8 at a ragged end) of them exist.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int n, float* v) {
  if (VEC) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 raw = *reinterpret_cast<const uint4*>(p);
      const T* t = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(t[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32<T>(p[i]) : 0.f;
  }
}

// Both kernels walk a grid of (8-column groups) x (rows): a block is TX groups wide and 256 / TX rows high, and each thread
// takes kU rows of its column, whose loads are in flight together. No division per element, and no two threads of a
// warp further apart than its columns.
constexpr int kU = 4;

// Four lanes own a block of 32 columns, eight columns each. The grid covers the padded scale array (rows to a
// multiple of 128, blocks to a multiple of 4), whose padding is written as zeros here.
// VEC: every 8-column group that exists is whole and 16-byte aligned.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_quantize_k(const T* __restrict__ x, uint8_t* __restrict__ codes,
                                                      uint8_t* __restrict__ scales, int64_t rows, int64_t cols,
                                                      int64_t ld, int64_t nkb, int txl) {
  const int64_t groups = nkb * 16;  // 8-column groups per padded row, a multiple of 16: quads of lanes are whole
  const int64_t g = ((int64_t)blockIdx.y << txl) + (threadIdx.x & ((1 << txl) - 1));
  const int64_t cb = (cols + kBlk - 1) / kBlk * 16;  // code bytes per row
  const int64_t c0 = g * 8;
  const int64_t row0 = ((int64_t)blockIdx.x * (256 >> txl) + (threadIdx.x >> txl)) * kU;
  const int n = (int)max((int64_t)0, min((int64_t)8, cols - c0));
  tc::pdl_wait();
  tc::pdl_trigger();
  float v[kU][8];
  const T* px = x + row0 * ld + c0;
#pragma unroll
  for (int u = 0; u < kU; ++u, px += ld) {
    if (row0 + u < rows && n > 0) {
      load8<T, VEC>(px, n, v[u]);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[u][k] = 0.f;
    }
  }
  const bool write_codes = c0 < cb * 2, write_scale = (g & 3) == 0 && g < groups;
  const int64_t padded = (rows + 127) / 128 * 128;
  uint8_t* pc = codes + row0 * cb + g * 4;
  uint8_t* ps = scales + scale_at(row0, g >> 2, nkb);  // kU rows share a group of 32: 16 bytes apart
#pragma unroll
  for (int u = 0; u < kU; ++u, pc += cb, ps += 16) {
    const bool in = row0 + u < rows;
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, magnitude_bits(v[u][k]));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t code = scale_code(top);
    if (in && write_codes) {
      const float inv = inverse_scale(code);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[u][k] *= inv;
      const uint32_t c = e2m1x8(v[u]);
      *reinterpret_cast<uint32_t*>(pc) = code == 255u ? 0u : c;
    }
    if (write_scale && row0 + u < padded) *ps = (in && n > 0) ? (uint8_t)code : (uint8_t)0;
  }
}

// Two floats -> two T, rounded to nearest.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) mx4_dequantize_k(const uint8_t* __restrict__ codes,
                                                        const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                        int64_t rows, int64_t cols, int64_t ld, int64_t nkb, int txl) {
  const int64_t g = ((int64_t)blockIdx.y << txl) + (threadIdx.x & ((1 << txl) - 1));
  const int64_t cb = (cols + kBlk - 1) / kBlk * 16;
  const int64_t row0 = ((int64_t)blockIdx.x * (256 >> txl) + (threadIdx.x >> txl)) * kU;
  const int n = (int)max((int64_t)0, min((int64_t)8, cols - g * 8));
  tc::pdl_wait();
  tc::pdl_trigger();
  if (n == 0) return;
  uint32_t c[kU], sc[kU];
  const uint8_t* pc = codes + row0 * cb + g * 4;
  const uint8_t* ps = scales + scale_at(row0, g >> 2, nkb);  // kU rows share a group of 32: 16 bytes apart
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    if (row0 + u < rows) {
      c[u] = *reinterpret_cast<const uint32_t*>(pc + u * cb);
      sc[u] = ps[16 * u];
    }
  }
  T* o = out + row0 * ld + g * 8;
#pragma unroll
  for (int u = 0; u < kU; ++u, o += ld) {
    if (row0 + u >= rows) break;
    const float s = e8m0_to_f32(sc[u]);
    __half2 h[4];
    e2m1x8_to_half2(c[u], h);
    float v[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float2 f = __half22float2(h[k]);
      v[2 * k] = f.x * s, v[2 * k + 1] = f.y * s;
    }
    if (VEC) {
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(o) = make_float4(v[0], v[1], v[2], v[3]);
        *(reinterpret_cast<float4*>(o) + 1) = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *reinterpret_cast<uint4*>(o) = make_uint4(pack_pair<T>(v[0], v[1]), pack_pair<T>(v[2], v[3]), pack_pair<T>(v[4], v[5]),
                                                  pack_pair<T>(v[6], v[7]));
      }
    } else {
      for (int k = 0; k < n; ++k) o[k] = from_f32<T>(v[k]);
    }
  }
}

// Block width (log2 of the 8-column groups, 16 to 256) and grid for `rows` x `groups`.
struct Walk {
  int txl;
  dim3 grid;
};
bool make_walk(int64_t rows, int64_t groups, Walk& w) {
  w.txl = 4;
  while (w.txl < 8 && (1ll << w.txl) < groups) ++w.txl;
  const int64_t gx = (rows + (256 >> w.txl) * kU - 1) / ((256 >> w.txl) * kU), gy = (groups + (1ll << w.txl) - 1) >> w.txl;
  if (gx >= (1ll << 31) || gy > 65535) return false;
  w.grid = dim3((unsigned)gx, (unsigned)gy);
  return true;
}

template <typename T>
int quantize_t(const b2_mx4_args* a, cudaStream_t st) {
  const int64_t nkb = (a->cols + 127) / 128;
  const bool vec = a->cols % 8 == 0 && ((uintptr_t)a->x & 15) == 0 && (a->ld * (int64_t)sizeof(T)) % 16 == 0;
  Walk w;
  if (!make_walk((a->rows + 127) / 128 * 128, nkb * 16, w)) return fail(B2_ERR_ARG, "mx4_quantize: matrix too large");
  return launch_pdl("mx4_quantize", vec ? mx4_quantize_k<T, true> : mx4_quantize_k<T, false>, w.grid, dim3(256), 0, st,
                    (const T*)a->x, a->codes, a->scales, a->rows, a->cols, a->ld, nkb, w.txl);
}

template <typename T>
int dequantize_t(const b2_mx4_args* a, cudaStream_t st) {
  const int64_t nkb = (a->cols + 127) / 128;
  const bool vec = a->cols % 8 == 0 && ((uintptr_t)a->out & 15) == 0 && (a->ld * (int64_t)sizeof(T)) % 16 == 0;
  Walk w;
  if (!make_walk(a->rows, (a->cols + 7) / 8, w)) return fail(B2_ERR_ARG, "mx4_dequantize: matrix too large");
  return launch_pdl("mx4_dequantize", vec ? mx4_dequantize_k<T, true> : mx4_dequantize_k<T, false>, w.grid, dim3(256), 0, st,
                    (const uint8_t*)a->codes, (const uint8_t*)a->scales, (T*)a->out, a->rows, a->cols, a->ld, nkb, w.txl);
}

int check(const b2_mx4_args* a, const void* data, const char* what) {
  if (!a) return fail(B2_ERR_ARG, std::string(what) + ": null arguments");
  if (a->rows < 0 || a->cols < 0) return fail(B2_ERR_ARG, std::string(what) + ": negative size");
  if (a->dtype != B2_F32 && a->dtype != B2_BF16 && a->dtype != B2_F16)
    return fail(B2_ERR_ARG, std::string(what) + ": dtype must be F32, BF16 or F16");
  if (a->rows == 0 || a->cols == 0) return 0;
  if (a->ld < a->cols && a->rows > 1) return fail(B2_ERR_ARG, std::string(what) + ": ld smaller than cols");
  if (!data || !a->codes || !a->scales) return fail(B2_ERR_ARG, std::string(what) + ": null pointer");
  if (((uintptr_t)a->codes | (uintptr_t)a->scales) & 15)
    return fail(B2_ERR_ARG, std::string(what) + ": codes and scales must be 16-byte aligned");
  if ((uintptr_t)data % dtype_size(a->dtype)) return fail(B2_ERR_ARG, std::string(what) + ": unaligned data pointer");
  return ensure_init();
}

}  // namespace
}  // namespace b2

extern "C" int64_t b2_mx4_code_bytes(int64_t cols) { return cols <= 0 ? 0 : (cols + 31) / 32 * 16; }
extern "C" int64_t b2_mx4_scale_bytes(int64_t rows, int64_t cols) {
  return rows <= 0 || cols <= 0 ? 0 : (rows + 127) / 128 * ((cols + 127) / 128) * 512;
}

extern "C" int b2_mx4_quantize(const b2_mx4_args* a, b2_stream_t stream) {
  using namespace b2;
  if (int rc = check(a, a ? a->x : nullptr, "mx4_quantize")) return rc;
  if (a->rows == 0 || a->cols == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case B2_F32: return quantize_t<float>(a, st);
    case B2_BF16: return quantize_t<__nv_bfloat16>(a, st);
    default: return quantize_t<__half>(a, st);
  }
}

extern "C" int b2_mx4_dequantize(const b2_mx4_args* a, b2_stream_t stream) {
  using namespace b2;
  if (int rc = check(a, a ? a->out : nullptr, "mx4_dequantize")) return rc;
  if (a->rows == 0 || a->cols == 0) return 0;
  cudaStream_t st = (cudaStream_t)stream;
  switch (a->dtype) {
    case B2_F32: return dequantize_t<float>(a, st);
    case B2_BF16: return dequantize_t<__nv_bfloat16>(a, st);
    default: return dequantize_t<__half>(a, st);
  }
}

// ---- product ------------------------------------------------------------------------------------------------------
// The tensor-core kernels of mx4_gemm.cu; dX reads W from the workspace, where it is expanded to bf16 first (exactly:
// every MXFP4 value that quantisation makes is a bf16 value).
namespace b2 {

bool mx4_gemm_tc_eligible(const b2_mx4_gemm_args* a);  // mx4_gemm.cu
int mx4_gemm_fwd(const b2_mx4_gemm_args* a, cudaStream_t st);
bool mx4_rows_eligible(const b2_mx4_gemm_args* a);     // mx4_rows.cu
int mx4_rows(const b2_mx4_gemm_args* a, cudaStream_t st);
int mx4_gemm_dx(const b2_mx4_gemm_args* a, const void* x, int64_t x_ld, const void* w, int64_t w_ld, cudaStream_t st);

namespace {

int64_t pad_to(int64_t k, int64_t m) { return (k + m - 1) / m * m; }
uint64_t up16(uint64_t v) { return (v + 15) / 16 * 16; }

int expand(const uint8_t* codes, const uint8_t* scales, void* out, int64_t rows, int64_t cols, int64_t ld, cudaStream_t st) {
  b2_mx4_args d{};
  d.codes = const_cast<uint8_t*>(codes), d.scales = const_cast<uint8_t*>(scales), d.out = out;
  d.rows = rows, d.cols = cols, d.ld = ld, d.dtype = B2_BF16;
  return b2_mx4_dequantize(&d, st);
}
int gemm_check(const b2_mx4_gemm_args* a) {
  if (!a) return fail(B2_ERR_ARG, "mx4_gemm: null arguments");
  if (a->M < 0 || a->N < 0 || a->K < 0) return fail(B2_ERR_ARG, "mx4_gemm: negative size");
  if (a->M == 0 || a->N == 0 || a->K == 0) return 0;
  if (!a->w_codes || !a->w_scales || !a->out || (a->transpose_w ? !a->x : !a->x && (!a->x_codes || !a->x_scales)))
    return fail(B2_ERR_ARG, "mx4_gemm: null pointer");
  if (((uintptr_t)a->w_codes | (uintptr_t)a->w_scales | (uintptr_t)a->x_codes | (uintptr_t)a->x_scales) & 15)
    return fail(B2_ERR_ARG, "mx4_gemm: codes and scales must be 16-byte aligned");
  if (a->out_ld < (a->transpose_w ? a->K : a->N)) return fail(B2_ERR_ARG, "mx4_gemm: out_ld smaller than a row");
  if (a->x && a->x_ld < (a->transpose_w ? a->N : a->K)) return fail(B2_ERR_ARG, "mx4_gemm: x_ld smaller than a row");
  if (!a->transpose_w && a->x && !mx4_rows_eligible(a))
    return fail(B2_ERR_ARG, "mx4_gemm: a forward with this many values of x takes them quantised");
  if (a->lora_r) {
    if (a->lora_r < 8 || a->lora_r > 64 || a->lora_r % 8 || !a->lora_h || !a->lora_b || a->lora_h_ld % 8 || a->lora_b_ld % 8 ||
        (((uintptr_t)a->lora_h | (uintptr_t)a->lora_b) & 15))
      return fail(B2_ERR_ARG, "mx4_gemm: lora_r must be 8..64 and a multiple of 8, with 16-byte aligned operands and rows");
  }
  return 0;
}

struct DxPlan {
  int64_t ldw, ldx;      // row strides of the expanded weight and of the copied dY
  bool copy_x;           // dY's rows are not whole 16-byte groups: copied into the workspace
  uint64_t x, bytes;     // offset of that copy; workspace bytes
};
DxPlan dx_plan(const b2_mx4_gemm_args* a) {
  DxPlan d;
  d.ldw = pad_to(a->K, 32), d.ldx = pad_to(a->N, 8);
  d.copy_x = a->x_ld % 8 || ((uintptr_t)a->x & 15);
  d.x = up16((uint64_t)a->N * d.ldw * 2);
  d.bytes = d.x + (d.copy_x ? (uint64_t)a->M * d.ldx * 2 : 0);
  return d;
}

}  // namespace
}  // namespace b2

extern "C" int b2_mx4_takes_x(int64_t M, int64_t N, int64_t K) {
  b2_mx4_gemm_args a{};
  a.M = M, a.N = N, a.K = K, a.x = &a;
  return b2::mx4_rows_eligible(&a) ? 1 : 0;
}

extern "C" uint64_t b2_mx4_gemm_workspace_bytes(const b2_mx4_gemm_args* a) {
  using namespace b2;
  if (!a || a->M <= 0 || a->N <= 0 || a->K <= 0 || !a->transpose_w) return 0;
  return dx_plan(a).bytes;
}

extern "C" int b2_mx4_gemm(const b2_mx4_gemm_args* a, b2_stream_t stream) {
  using namespace b2;
  if (int rc = gemm_check(a)) return rc;
  if (a->M == 0 || a->N == 0 || a->K == 0) return 0;
  if (int rc = ensure_init()) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  if (!mx4_gemm_tc_eligible(a)) return fail(B2_ERR_ARG, "mx4_gemm: sizes beyond 2^30, or no sm_100a device");
  if (!a->transpose_w) return a->x ? mx4_rows(a, st) : mx4_gemm_fwd(a, st);
  if (!a->workspace || ((uintptr_t)a->workspace & 15))
    return fail(B2_ERR_ARG, "mx4_gemm: a 16-byte aligned workspace of b2_mx4_gemm_workspace_bytes() is required");
  const DxPlan d = dx_plan(a);
  if (int rc = expand(a->w_codes, a->w_scales, a->workspace, a->N, d.ldw, d.ldw, st)) return rc;
  const void* x = a->x;
  if (d.copy_x) {
    void* xc = (char*)a->workspace + d.x;
    if (int rc = check_cuda(cudaMemcpy2DAsync(xc, d.ldx * 2, a->x, a->x_ld * 2, a->N * 2, a->M, cudaMemcpyDeviceToDevice, st),
                            "mx4_gemm copy"))
      return rc;
    x = xc;
  }
  return mx4_gemm_dx(a, x, d.copy_x ? d.ldx : a->x_ld, a->workspace, d.ldw, st);
}
