// Rows to few bits: quantize_fp4, rmsnorm_quantize and their inverses.
//
//   h = x + residual,  y = h * (1/sqrt(mean(h^2) + eps)) * weight     (norm only)
//   z = group Hadamard of y                                           (optional)
//   int8:  s = max(amax(z)/127, 1e-30),  code = round-half-away(z * (1/s))
//   mxfp4: per 32, s = 2^(floor(log2 amax) - 2), code = E2M1(z / s)
//   nvfp4: g = max(amax(row)/2688, 1e-30); per 16, s = E4M3(amax/(6g)), code = E2M1(z * (1/(s*g)))
//
// A row is spread over TPR threads, 16 consecutive columns ("a chunk") to a
// lane, which is one nvfp4 block, half an mxfp4 block, and the unit of the
// register Hadamard.  The row stays in registers from the load to the codes
// (CH chunks per thread), so HBM sees each input once and each output once;
// rows too long for that are read again for each reduction (CH = 0), from L2.
// The sum of squares is held in 64 bits, so the norm does not depend on the
// order of its sum and codes next to a rounding border are reproducible.
#include <cuda_fp8.h>

#include "hadamard.cuh"
#include "internal.h"
#include "lowp.cuh"

namespace ic {
namespace {

struct RowArgs {
  const void* x;
  const void* residual;
  const void* weight;
  void* residual_out;
  int64_t M, K, kp;  // rows, input columns, held columns
  int64_t ldx, ldr, ldo;
  int wdtype;
  float eps;
  int rot;
  const float* row_scale_in;  // nvfp4 with given row scales (stride 0 or 1), or null
  int64_t rs_stride;
  void* q;      // int8 codes or packed 4-bit codes
  int64_t ldq;  // bytes per row of q
  uint8_t* scales;
  int64_t ktiles;
  float* row_scale;
  int32_t* sums;
  int tpr;
};

// 16 elements from p; elements at or beyond `left` read as zero
template <typename T>
__device__ __forceinline__ void load16(const T* p, int64_t left, float (&v)[16]) {
  constexpr int V = 16 / sizeof(T);
  if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    uint4 raw[16 / V];
#pragma unroll
    for (int i = 0; i < 16 / V; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
#pragma unroll
    for (int i = 0; i < 16 / V; ++i) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
#pragma unroll
      for (int u = 0; u < V; ++u) v[i * V + u] = load_as_f32(e + u);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = j < left ? load_as_f32(p + j) : 0.f;
  }
}

__device__ __forceinline__ void load16_any(const void* p, int dtype, int64_t at, int64_t left, float (&v)[16]) {
  if (dtype == IC_F32) load16(static_cast<const float*>(p) + at, left, v);
  else if (dtype == IC_F16) load16(static_cast<const __half*>(p) + at, left, v);
  else load16(static_cast<const __nv_bfloat16*>(p) + at, left, v);
}

template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ void store16(T* p, int64_t left, const float (&v)[16]) {
  constexpr int V = 16 / sizeof(T);
  if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 16 / V; ++i) {
      uint4 raw;
      T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int u = 0; u < V; ++u) e[u] = from_f32<T>(v[i * V + u]);
      reinterpret_cast<uint4*>(p)[i] = raw;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j < left) p[j] = from_f32<T>(v[j]);
  }
}

// |x| as ordered bits: NaN above infinity above every finite value
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr unsigned INF_BITS = 0x7f800000u;

__device__ __forceinline__ unsigned amax16(const float (&v)[16]) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < 16; ++j) m = max(m, abs_bits(v[j]));
  return m;
}

// 8 fp32 values -> 8 E2M1 codes (round to nearest even, saturating), element 0 in the low nibble
__device__ __forceinline__ uint32_t e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n .reg .b8 b0, b1, b2, b3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
      " cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
      " mov.b32 %0, {b0, b1, b2, b3};\n}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ uint32_t to_e4m3(float x) {
  return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ float from_e4m3(uint32_t b) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E4M3)));
}

// reductions over the TPR threads of a row (TPR a multiple of 32); `buf` holds
// one value per warp of the CTA
template <typename V, typename F>
__device__ __forceinline__ V row_reduce(V v, int tpr, V* buf, F op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr == 32) return v;
  const int w = threadIdx.x >> 5, nw = tpr >> 5, w0 = w & ~(nw - 1);
  __syncthreads();  // buf may still be read from the last reduction
  if ((threadIdx.x & 31) == 0) buf[w] = v;
  __syncthreads();
  v = buf[w0];
  for (int i = 1; i < nw; ++i) v = op(v, buf[w0 + i]);
  return v;
}

// what the row's codes are formed with
struct RowScale {
  float s;    // int8: reciprocal of the row's scale; nvfp4: g
  float i6g;  // nvfp4: 1 / (6 g)
  bool bad;   // a value of the row is not finite: codes 0
};

template <int FMT>
__device__ __forceinline__ int emit_chunk(const RowArgs& a, int64_t row, int64_t c, int64_t nch, float (&v)[16],
                                          const RowScale& rs) {
  const int lane = threadIdx.x & 31;
  const bool live = row < a.M && c < nch;
  if (FMT == IC_INT8) {
    uint32_t w[4];
    int sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float y = rs.bad ? 0.f : rhaz(__fmul_rn(v[4 * i + u], rs.s));
        const int code = (int)fminf(fmaxf(y, -128.f), 127.f);
        sum += code;
        w[i] |= (uint32_t)(code & 255) << (8 * u);
      }
    }
    if (live) *reinterpret_cast<uint4*>(static_cast<int8_t*>(a.q) + row * a.ldq + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    return live ? sum : 0;
  }
  uint32_t byte;
  float inv;
  bool bad;
  unsigned m = amax16(v);
  if (FMT == IC_MXFP4) {
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));  // the block is this chunk and its neighbour
    bad = m >= INF_BITS;
    const uint32_t e = m >> 23;
    byte = bad ? 255u : (e > 2 ? e - 2 : 0u);
    inv = bad ? 0.f : __uint_as_float((254u - byte) << 23);
  } else {
    bad = m >= INF_BITS || rs.bad;
    byte = bad ? (rs.bad ? 0u : 0x7fu) : to_e4m3(__fmul_rn(__uint_as_float(m), rs.i6g));
    const float s = from_e4m3(byte);
    inv = bad || byte == 0 ? 0.f : __fdiv_rn(1.f, __fmul_rn(s, rs.s));
  }
  float y[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) y[j] = bad ? 0.f : __fmul_rn(v[j], inv);
  const uint2 codes = make_uint2(e2m1x8(y), e2m1x8(y + 8));
  if (live) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.q) + row * a.ldq + c * 8) = codes;
  // four blocks' bytes to one word
  uint32_t word;
  int64_t kt;
  bool first;
  if (FMT == IC_MXFP4) {
    word = byte << (8 * ((lane >> 1) & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    kt = c >> 3;
    first = (lane & 7) == 0;
  } else {
    word = byte << (8 * (lane & 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 1);
    word |= __shfl_xor_sync(0xffffffffu, word, 2);
    kt = c >> 2;
    first = (lane & 3) == 0;
  }
  if (first && kt < a.ktiles) *reinterpret_cast<uint32_t*>(a.scales + scale_word(row, kt, a.ktiles)) = word;
  return 0;
}

// h = x + residual of one chunk, optionally written to residual_out
template <typename T, bool NORM>
__device__ __forceinline__ void load_chunk(const RowArgs& a, int64_t row, int64_t c, float (&v)[16], bool write) {
  const int64_t left = row < a.M ? a.K - c * 16 : 0;
  load16(static_cast<const T*>(a.x) + (left > 0 ? row * a.ldx + c * 16 : 0), left, v);
  if (NORM && a.residual) {
    float r[16];
    load16(static_cast<const T*>(a.residual) + (left > 0 ? row * a.ldr + c * 16 : 0), left, r);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fadd_rn(v[j], r[j]);
    // the stream's value is rounded to its type here; the norm goes on from the sum in 32 bits
    if (write && left > 0) store16(static_cast<T*>(a.residual_out) + row * a.ldo + c * 16, left, v);
  }
}

template <bool NORM>
__device__ __forceinline__ void finish_chunk(const RowArgs& a, int64_t c, float (&v)[16], float rstd, int l) {
  if (NORM) {
    float w[16];
    load16_any(a.weight, a.wdtype, a.K - c * 16 > 0 ? c * 16 : 0, a.K - c * 16, w);
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = __fmul_rn(__fmul_rn(v[j], rstd), w[j]);
  }
  if (a.rot) hadamard_regs16(v, a.rot, l);
}

template <typename T, int FMT, bool NORM, int CH>
__global__ void __launch_bounds__(512) rows_kernel(const RowArgs a) {
  __shared__ double buf[32];
  const int tpr = a.tpr, t = threadIdx.x & (tpr - 1);
  const int64_t row = (int64_t)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const int64_t nch = cdiv(a.kp, 16);
  const int l = a.rot ? (threadIdx.x & (a.rot / 16 - 1)) : 0;  // this lane's chunk of its rotation group
  const int n = CH ? CH : (int)cdiv(nch, tpr);
  constexpr bool NEED_AMAX = FMT == IC_INT8 || FMT == IC_NVFP4;
  float v[CH ? CH : 1][16];
  float rstd = 0.f;
  if (CH) {
#pragma unroll
    for (int i = 0; i < CH; ++i) load_chunk<T, NORM>(a, row, (int64_t)i * tpr + t, v[i], true);
  }
  if (NORM) {
    double ss = 0.0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      if (!CH) load_chunk<T, NORM>(a, row, (int64_t)i * tpr + t, v[0], true);
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const double d = v[CH ? i : 0][j];
        ss = fma(d, d, ss);
      }
    }
    ss = row_reduce(ss, tpr, buf, [](double p, double q) { return p + q; });
    // squares of fp32 values cannot overflow here: an infinite sum is an infinite input, which marks the whole row
    rstd = isfinite(ss) ? (float)(1.0 / sqrt(ss / (double)a.K + (double)a.eps)) : __int_as_float(0x7fc00000);
  }
  if (CH) {
#pragma unroll
    for (int i = 0; i < CH; ++i) finish_chunk<NORM>(a, (int64_t)i * tpr + t, v[i], rstd, l);
  }
  RowScale rs{0.f, 0.f, false};
  if (NEED_AMAX) {
    unsigned m = 0;
    if (!a.row_scale_in) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        if (!CH) {
          load_chunk<T, NORM>(a, row, (int64_t)i * tpr + t, v[0], false);
          finish_chunk<NORM>(a, (int64_t)i * tpr + t, v[0], rstd, l);
        }
        m = max(m, amax16(v[CH ? i : 0]));
      }
      m = row_reduce(m, tpr, reinterpret_cast<unsigned*>(buf), [](unsigned p, unsigned q) { return max(p, q); });
    }
    float s;
    if (FMT == IC_INT8) {
      rs.bad = m >= INF_BITS;
      s = fmaxf(__fmul_rn(__uint_as_float(m), (float)(1.0 / 127.0)), LOWP_SCALE_FLOOR);
      rs.s = __fdiv_rn(1.f, s);
    } else {
      if (a.row_scale_in) {
        s = row < a.M ? a.row_scale_in[row * a.rs_stride] : 1.f;
        rs.bad = !(s > 0.f) || abs_bits(s) >= INF_BITS;
      } else {
        rs.bad = m >= INF_BITS;
        s = fmaxf(__fmul_rn(__uint_as_float(m), (float)(1.0 / 2688.0)), LOWP_SCALE_FLOOR);
      }
      rs.s = s;
      rs.i6g = __fdiv_rn(1.f, __fmul_rn(6.f, s));
    }
    if (t == 0 && row < a.M) a.row_scale[row] = rs.bad ? __uint_as_float(0x7fc00000u) : s;
  }
  int sum = 0;
#pragma unroll
  for (int i = 0; i < n; ++i) {
    if (!CH) {
      load_chunk<T, NORM>(a, row, (int64_t)i * tpr + t, v[0], false);
      finish_chunk<NORM>(a, (int64_t)i * tpr + t, v[0], rstd, l);
    }
    sum += emit_chunk<FMT>(a, row, (int64_t)i * tpr + t, nch, v[CH ? i : 0], rs);
  }
  if (FMT == IC_INT8 && a.sums) {
    sum = row_reduce(sum, tpr, reinterpret_cast<int*>(buf), [](int p, int q) { return p + q; });
    if (t == 0 && row < a.M) a.sums[row] = sum;
  }
}

template <typename T, int FMT, bool NORM>
int launch_rows(RowArgs a, cudaStream_t st) {
  const int64_t nch = cdiv(a.kp, 16);
  // one chunk per thread up to 256 threads, then more chunks per thread
  int tpr = 32;
  while (tpr < 256 && tpr < nch) tpr *= 2;
  int ch = (int)cdiv(nch, tpr);
  if (ch > 4) {
    tpr = 512;
    ch = (int)cdiv(nch, tpr);
  }
  a.tpr = tpr;
  const int threads = std::max(tpr, 128);
  const int rpc = threads / tpr;
  // the 4-bit formats' scale tiles hold 128 rows: the grid covers the padding rows too
  const int64_t rows = FMT == IC_INT8 ? a.M : cdiv(a.M, 128) * 128;
  const int64_t grid = cdiv(rows, rpc);
  if (grid > INT32_MAX) return fail(IC_ERR_UNSUPPORTED, "quantize: too many rows");
  if (ch <= 1) rows_kernel<T, FMT, NORM, 1><<<(unsigned)grid, threads, 0, st>>>(a);
  else if (ch <= 2) rows_kernel<T, FMT, NORM, 2><<<(unsigned)grid, threads, 0, st>>>(a);
  else if (ch <= 4) rows_kernel<T, FMT, NORM, 4><<<(unsigned)grid, threads, 0, st>>>(a);
  else rows_kernel<T, FMT, NORM, 0><<<(unsigned)grid, threads, 0, st>>>(a);
  IC_CHECK_LAUNCH();
  return IC_OK;
}

template <typename T>
int dispatch_rows(const RowArgs& a, int fmt, bool norm, cudaStream_t st) {
  if (norm) {
    if (fmt == IC_INT8) return launch_rows<T, IC_INT8, true>(a, st);
    if (fmt == IC_MXFP4) return launch_rows<T, IC_MXFP4, true>(a, st);
    return launch_rows<T, IC_NVFP4, true>(a, st);
  }
  if (fmt == IC_MXFP4) return launch_rows<T, IC_MXFP4, false>(a, st);
  return launch_rows<T, IC_NVFP4, false>(a, st);
}

int dispatch_rows(const RowArgs& a, int dtype, int fmt, bool norm, cudaStream_t st) {
  switch (dtype) {
    case IC_F32: return dispatch_rows<float>(a, fmt, norm, st);
    case IC_F16: return dispatch_rows<__half>(a, fmt, norm, st);
    default: return dispatch_rows<__nv_bfloat16>(a, fmt, norm, st);
  }
}

// checks shared by the two quantizers; what: the entry point's name
int check_rows(const char* what, const RowArgs& a, int dtype, int fmt) {
  if (a.M < 0 || a.K <= 0 || a.ldx < a.K) return fail(IC_ERR_INVALID, "%s: bad shape", what);
  if (a.K > (int64_t(1) << 24)) return fail(IC_ERR_UNSUPPORTED, "%s: rows longer than 2^24", what);
  if (dtype < IC_F32 || dtype > IC_BF16) return fail(IC_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (a.rot != 0 && !hadamard_regs_ok(a.rot))
    return fail(IC_ERR_INVALID, "%s: rot must be 0 or a power of two in 16..512, got %d", what, a.rot);
  const int64_t unit = std::max<int64_t>(fmt == IC_INT8 ? 1 : 32, a.rot);
  if (a.kp != cdiv(a.K, unit) * unit) return fail(IC_ERR_INVALID, "%s: kp must be K rounded up to a multiple of %lld", what, (long long)unit);
  const int64_t need = fmt == IC_INT8 ? cdiv(a.kp, 16) * 16 : a.kp / 2;
  if (a.ldq < need || a.ldq % 16) return fail(IC_ERR_INVALID, "%s: rows of codes need a pitch of at least %lld bytes, a multiple of 16", what, (long long)need);
  if (a.M > 0 && (!a.x || !a.q || (fmt != IC_INT8 && !a.scales) || (fmt != IC_MXFP4 && !a.row_scale)))
    return fail(IC_ERR_INVALID, "%s: null pointer", what);
  if ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.scales)) & 15)
    return fail(IC_ERR_INVALID, "%s: codes and scales must be 16-byte aligned", what);
  return IC_OK;
}

// ---------------------------------------------------------------- dequantize
template <typename T, int FMT>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* __restrict__ q, int64_t ldq, int64_t M, int64_t kp,
                                                      const uint8_t* __restrict__ scales, int64_t ktiles,
                                                      const float* __restrict__ row_scale, T* __restrict__ out,
                                                      int64_t ldo) {
  const int64_t nch = cdiv(kp, 16);
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  const int64_t row = i / nch, c = i - row * nch;
  if (row >= M) return;
  float v[16];
  if (FMT == IC_INT8) {
    const float s = row_scale[row];
    const int8_t* p = reinterpret_cast<const int8_t*>(q) + row * ldq + c * 16;
    const int64_t left = kp - c * 16;
    if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
      const uint4 raw = *reinterpret_cast<const uint4*>(p);
      const int8_t* e = reinterpret_cast<const int8_t*>(&raw);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = __fmul_rn((float)e[j], s);
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = j < left ? __fmul_rn((float)p[j], s) : 0.f;
    }
  } else {
    const int64_t b = FMT == IC_MXFP4 ? c >> 1 : c;
    const uint32_t byte = scales[scale_word(row, b >> 2, ktiles) + (b & 3)];
    const float s = FMT == IC_MXFP4 ? (byte == 255u ? __uint_as_float(0x7fc00000u)
                                                    : __uint_as_float(byte ? byte << 23 : 0x00400000u))
                                    : from_e4m3(byte);
    const float g = FMT == IC_NVFP4 ? row_scale[row] : 1.f;
    const uint2 raw = *reinterpret_cast<const uint2*>(q + row * ldq + c * 8);
    const uint32_t w[2] = {raw.x, raw.y};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t code = (w[j >> 3] >> (4 * (j & 7))) & 15u;
      const uint32_t e = (code >> 1) & 3u, f = code & 1u;
      // E2M1: 0, 0.5 below 1, else (1 + f/2) 2^(e-1)
      float x = e ? __uint_as_float(((126u + e) << 23) | (f << 22)) : (f ? 0.5f : 0.f);
      x = code & 8u ? -x : x;
      v[j] = __fmul_rn(x, s);
      if (FMT == IC_NVFP4) v[j] = __fmul_rn(v[j], g);
    }
  }
  store16(out + row * ldo + c * 16, kp - c * 16, v);
}

template <int FMT>
int launch_dequant(const void* q, int64_t ldq, int64_t M, int64_t kp, const uint8_t* scales, int64_t ktiles,
                   const float* row_scale, int dtype, void* out, int64_t ldo, cudaStream_t st) {
  const uint8_t* p = static_cast<const uint8_t*>(q);
  const int64_t grid = cdiv(M * cdiv(kp, 16), 256);
  if (grid > INT32_MAX) return fail(IC_ERR_UNSUPPORTED, "dequantize: too many elements");
  switch (dtype) {
    case IC_F32: dequant_kernel<float, FMT><<<(unsigned)grid, 256, 0, st>>>(p, ldq, M, kp, scales, ktiles, row_scale, (float*)out, ldo); break;
    case IC_F16: dequant_kernel<__half, FMT><<<(unsigned)grid, 256, 0, st>>>(p, ldq, M, kp, scales, ktiles, row_scale, (__half*)out, ldo); break;
    case IC_BF16: dequant_kernel<__nv_bfloat16, FMT><<<(unsigned)grid, 256, 0, st>>>(p, ldq, M, kp, scales, ktiles, row_scale, (__nv_bfloat16*)out, ldo); break;
    default: return fail(IC_ERR_INVALID, "dequantize: unknown dtype %d", dtype);
  }
  IC_CHECK_LAUNCH();
  return IC_OK;
}

__global__ void __launch_bounds__(256) row_sums_kernel(const int8_t* __restrict__ q, int64_t ldq, int64_t M, int64_t K,
                                                       int32_t* __restrict__ sums) {
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= M) return;
  int s = 0;
  for (int64_t k = threadIdx.x & 31; k < K; k += 32) s += q[row * ldq + k];
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) sums[row] = s;
}

}  // namespace
}  // namespace ic

extern "C" int ic_fp4_quantize(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, int fmt, int rot,
                               int64_t kp, const float* row_scale_in, int64_t row_scale_stride, uint8_t* packed,
                               uint8_t* scales, float* row_scale, void* stream) {
  using namespace ic;
  if (fmt != IC_MXFP4 && fmt != IC_NVFP4) return fail(IC_ERR_INVALID, "fp4_quantize: unknown format %d", fmt);
  if (row_scale_in && (fmt != IC_NVFP4 || row_scale_stride < 0 || row_scale_stride > 1))
    return fail(IC_ERR_INVALID, "fp4_quantize: given row scales are for nvfp4, with stride 0 or 1");
  RowArgs a{};
  a.x = x, a.M = M, a.K = K, a.kp = kp, a.ldx = ldx, a.rot = rot;
  a.row_scale_in = row_scale_in, a.rs_stride = row_scale_stride;
  a.q = packed, a.ldq = kp / 2, a.scales = scales, a.ktiles = fp4_ktiles(fmt, kp), a.row_scale = row_scale;
  IC_TRY(check_rows("fp4_quantize", a, dtype, fmt));
  if (M == 0) return IC_OK;
  return dispatch_rows(a, dtype, fmt, false, (cudaStream_t)stream);
}

extern "C" int ic_rmsnorm_quantize(const void* x, const void* residual, int dtype, int64_t M, int64_t K, int64_t ldx,
                                   int64_t ldr, const void* weight, int weight_dtype, float eps, int fmt, int rot,
                                   int64_t kp, void* residual_out, int64_t ldo, void* q, int64_t ldq, uint8_t* scales,
                                   float* row_scale, int32_t* sums, void* stream) {
  using namespace ic;
  if (fmt != IC_INT8 && fmt != IC_MXFP4 && fmt != IC_NVFP4)
    return fail(IC_ERR_INVALID, "rmsnorm_quantize: unknown format %d", fmt);
  if (weight_dtype < IC_F32 || weight_dtype > IC_BF16)
    return fail(IC_ERR_INVALID, "rmsnorm_quantize: unknown weight dtype %d", weight_dtype);
  if (!(eps >= 0.f)) return fail(IC_ERR_INVALID, "rmsnorm_quantize: eps must not be negative");
  RowArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.residual_out = residual_out;
  a.M = M, a.K = K, a.kp = kp, a.ldx = ldx, a.ldr = ldr, a.ldo = ldo, a.wdtype = weight_dtype, a.eps = eps, a.rot = rot;
  a.q = q, a.ldq = ldq, a.scales = scales, a.row_scale = row_scale, a.sums = sums;
  a.ktiles = fmt == IC_INT8 ? 0 : fp4_ktiles(fmt, kp);
  IC_TRY(check_rows("rmsnorm_quantize", a, dtype, fmt));
  if (M > 0 && !weight) return fail(IC_ERR_INVALID, "rmsnorm_quantize: null weight");
  if (M > 0 && residual && (!residual_out || ldr < K || ldo < K))
    return fail(IC_ERR_INVALID, "rmsnorm_quantize: a residual needs residual_out and row pitches of at least K");
  if (residual && (residual_out == x || residual_out == residual))
    return fail(IC_ERR_INVALID, "rmsnorm_quantize: residual_out must not overlap x or residual");
  if (M == 0) return IC_OK;
  return dispatch_rows(a, dtype, fmt, true, (cudaStream_t)stream);
}

extern "C" int ic_fp4_dequantize(const uint8_t* packed, const uint8_t* scales, const float* row_scale, int fmt,
                                 int64_t M, int64_t kp, int dtype, void* out, int64_t ldo, void* stream) {
  using namespace ic;
  if (fmt != IC_MXFP4 && fmt != IC_NVFP4) return fail(IC_ERR_INVALID, "fp4_dequantize: unknown format %d", fmt);
  if (M < 0 || kp < 0 || kp % 32 || ldo < kp) return fail(IC_ERR_INVALID, "fp4_dequantize: bad shape");
  if (M == 0 || kp == 0) return IC_OK;
  if (!packed || !scales || !out || (fmt == IC_NVFP4 && !row_scale))
    return fail(IC_ERR_INVALID, "fp4_dequantize: null pointer");
  if (reinterpret_cast<uintptr_t>(packed) & 7) return fail(IC_ERR_INVALID, "fp4_dequantize: codes must be 8-byte aligned");
  const int64_t kt = fp4_ktiles(fmt, kp);
  if (fmt == IC_MXFP4) return launch_dequant<IC_MXFP4>(packed, kp / 2, M, kp, scales, kt, row_scale, dtype, out, ldo, (cudaStream_t)stream);
  return launch_dequant<IC_NVFP4>(packed, kp / 2, M, kp, scales, kt, row_scale, dtype, out, ldo, (cudaStream_t)stream);
}

extern "C" int ic_int8_dequantize(const int8_t* codes, int64_t ldq, const float* row_scale, int64_t M, int64_t K,
                                  int dtype, void* out, int64_t ldo, void* stream) {
  using namespace ic;
  if (M < 0 || K < 0 || ldq < K || ldo < K) return fail(IC_ERR_INVALID, "int8_dequantize: bad shape");
  if (M == 0 || K == 0) return IC_OK;
  if (!codes || !row_scale || !out) return fail(IC_ERR_INVALID, "int8_dequantize: null pointer");
  return launch_dequant<IC_INT8>(codes, ldq, M, K, nullptr, 0, row_scale, dtype, out, ldo, (cudaStream_t)stream);
}

extern "C" int ic_int8_row_sums(const int8_t* codes, int64_t ldq, int64_t M, int64_t K, int32_t* sums, void* stream) {
  using namespace ic;
  if (M < 0 || K < 0 || ldq < K) return fail(IC_ERR_INVALID, "int8_row_sums: bad shape");
  if (M == 0) return IC_OK;
  if (!sums || (K > 0 && !codes)) return fail(IC_ERR_INVALID, "int8_row_sums: null pointer");
  if (cdiv(M, 8) > INT32_MAX) return fail(IC_ERR_UNSUPPORTED, "int8_row_sums: too many rows");
  row_sums_kernel<<<(unsigned)cdiv(M, 8), 256, 0, (cudaStream_t)stream>>>(codes, ldq, M, K, sums);
  IC_CHECK_LAUNCH();
  return IC_OK;
}
