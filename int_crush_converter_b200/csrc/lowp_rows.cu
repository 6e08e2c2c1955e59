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
// register Hadamard.  Chunks are held two at a time as fp32 pairs (chunk A in
// the low halves, chunk B, TPR chunks on, in the high ones), so additions and
// products of both are one packed .f32x2 instruction.  The row stays in
// registers from the load to the codes (NP pairs per thread), so HBM sees each
// input once and each output once; rows too long for that are read again for
// each reduction (NP = 0), from L2.  Resident CTAs take rows by turns and load
// the next ones while they work on these.
//
// What bounds them, measured on B200 (copy rate 6.56 TB/s), calls back to back with the
// one or two microseconds between them:
//   quantize 16384 x 4096 bf16   mxfp4 31 us (HBM: 5.5 TB/s), nvfp4 35 us (the row's maximum
//                                between two barriers), nvfp4 rot256 61 us (two transposes move
//                                16 bytes an element: 70% of shared memory's wavefronts, with 60%
//                                of the issue slots and 32% of the warps; none of them a limit)
//   norm 4608 x 4096 bf16 with residual   mxfp4 28 us (4.4 TB/s), int8 33 us, nvfp4 rot256 39 us
//   dequantize 16384 x 4096 nvfp4 to bf16 32 us (5.4 TB/s); one row of 4096: norm 4.5 us in a graph
//   norm 1000 x 12288 bf16 with residual  int8 41 us, mxfp4 rot256 58 us: the instances of the norm
//                                for 8192 < K <= 32768 spill 0.7 to 4 KB a thread
// Packed arithmetic, three-input maxima and the transpose are there because the
// first kernels were bound by instruction issue (80% of the slots, 43
// instructions an element: 98 us for the rotated nvfp4 case).
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
  int tpr;         // threads per row
  int tshift, tmask;  // row within the CTA = thread >> tshift, thread within the row = thread & tmask
  int64_t groups;  // row groups, blockDim.x / tpr rows each
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

// whole 32-byte sectors per lane
__device__ __forceinline__ void load32(const void* p, uint4& a, uint4& b) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a.x), "=r"(a.y), "=r"(a.z), "=r"(a.w), "=r"(b.x), "=r"(b.y), "=r"(b.z), "=r"(b.w)
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w),
               "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

template <typename T>
__device__ __forceinline__ void store16(T* p, int64_t left, const float (&v)[16]) {
  constexpr int V = 16 / sizeof(T);
  if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
    uint4 raw[16 / V];
#pragma unroll
    for (int i = 0; i < 16 / V; ++i) {
      T* e = reinterpret_cast<T*>(&raw[i]);
#pragma unroll
      for (int u = 0; u < V; ++u) e[u] = from_f32<T>(v[i * V + u]);
    }
#pragma unroll
    for (int i = 0; i < 16 / V; i += 2) store32(p + i * V, raw[i], raw[i + 1]);
  } else if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
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

constexpr unsigned INF_BITS = 0x7f800000u;  // |x| as bits: NaN above infinity above every finite value

// max(|a|, |b|, |c|), NaN if one is
__device__ __forceinline__ float amax3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// bits of the largest magnitude of a chunk
__device__ __forceinline__ unsigned amax16(const float (&v)[16]) {
  const float a = amax3(v[0], v[1], v[2]), b = amax3(v[3], v[4], v[5]), c = amax3(v[6], v[7], v[8]),
              d = amax3(v[9], v[10], v[11]), e = amax3(v[12], v[13], v[14]);
  return __float_as_uint(amax3(amax3(a, b, c), amax3(d, e, v[15]), 0.f));
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
// four values, each x + (x < 0 ? -1/2 : 1/2) towards zero (rhaz, for magnitudes within int8 and a
// half), saturated to int8 codes, value 0 in the low byte
__device__ __forceinline__ uint32_t int8x4(float a, float b, float c, float d) {
  auto r = [](float x) { return __float2int_rz(__fadd_rn(x, copysignf(0.5f, x))); };
  uint32_t w;
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(w) : "r"(r(d)), "r"(r(c)));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %0;" : "+r"(w) : "r"(r(b)), "r"(r(a)));
  return w;
}

// reductions over the TPR threads of a row (TPR a multiple of 32, and a power of
// two where a CTA has several rows); `buf` holds one value per warp of the CTA
template <typename V, typename F>
__device__ __forceinline__ V row_reduce(V v, int tpr, int tmask, V* buf, F op) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (tpr == 32) return v;
  const int w = threadIdx.x >> 5, nw = tpr >> 5, w0 = w & ~(tmask >> 5);
  __syncthreads();  // buf may still be read from the last reduction
  if ((threadIdx.x & 31) == 0) buf[w] = v;
  __syncthreads();
  v = buf[w0];
  for (int i = 1; i < nw; ++i) v = op(v, buf[w0 + i]);
  return v;
}

// ------------------------------------------------------------ packed Hadamard
// The stages of hadamard_regs16 (same order, same fp32 operations) on pairs.
__device__ __forceinline__ void h4_pair(f2& x0, f2& x1, f2& x2, f2& x3) {
  const f2 p = add2(x0, x1), m = sub2(x0, x1), P = add2(x2, x3), M = sub2(x2, x3);
  x0 = add2(p, M);
  x1 = sub2(p, M);
  x2 = add2(m, P);
  x3 = sub2(P, m);
}
__device__ __forceinline__ void two_digits(f2 (&v)[16]) {
#pragma unroll
  for (int q = 0; q < 4; ++q) h4_pair(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
#pragma unroll
  for (int q = 0; q < 4; ++q) h4_pair(v[q], v[4 + q], v[8 + q], v[12 + q]);
}
__device__ __forceinline__ f2 shfl2(f2 x, int m) {
  return pk2(__shfl_xor_sync(0xffffffffu, lo2(x), m), __shfl_xor_sync(0xffffffffu, hi2(x), m));
}

constexpr int TEAM_BYTES = 16 * 136;  // 16 rows of 16 pairs, 8 bytes apart from a multiple of the banks

// rot = 256: both lane digits after one transpose of the team's 16 x 16 pairs
__device__ __forceinline__ void hadamard256(f2 (&v)[16], unsigned char* team, int l) {
  two_digits(v);
#pragma unroll
  for (int e = 0; e < 16; ++e) *reinterpret_cast<f2*>(team + l * 136 + e * 8) = v[e];
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = *reinterpret_cast<const f2*>(team + e * 136 + l * 8);
  two_digits(v);
  const f2 scale = pk2(0.0625f, 0.0625f);
#pragma unroll
  for (int e = 0; e < 16; ++e) *reinterpret_cast<f2*>(team + e * 136 + l * 8) = mul2(v[e], scale);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < 16; ++e) v[e] = *reinterpret_cast<const f2*>(team + l * 136 + e * 8);
  __syncwarp();
}

// other group sizes: lane digits by shuffles
__device__ __forceinline__ void hadamard_pair(f2 (&v)[16], int rot, int l) {
  const int L = rot / 16;
  if (is_pow4(rot)) {
    two_digits(v);
    float scale = 0.25f;
    for (int m = 1; m < L; m <<= 2) {
      // output k is (a_k + a_{k^1}) + (a_{k^2} - a_{k^3}): the difference comes whole from lane k^2
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const f2 o = shfl2(v[j], m);
        v[j] = add2(add2(v[j], o), shfl2(sub2(v[j], o), 2 * m));
      }
      scale *= 0.5f;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = mul2(v[j], pk2(scale, scale));
  } else {
#pragma unroll
    for (int st = 1; st < 16; st <<= 1) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (j & st) continue;
        const f2 a0 = v[j], a1 = v[j + st];
        v[j] = add2(a0, a1);
        v[j + st] = sub2(a0, a1);
      }
    }
    for (int m = 1; m < L; m <<= 1) {
      // the lower lane takes a + b, the upper a - b: its own value times 1 or -1, exactly, plus the other's
      const float sign = (l & m) != 0 ? -1.f : 1.f;
      const f2 own = pk2(sign, sign);
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = fma2(v[j], own, shfl2(v[j], m));
    }
    const float c = (float)(1.0 / sqrt((double)rot));  // fp32(1/sqrt(n)), rotation.py:36
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = mul2(v[j], pk2(c, c));
  }
}

// what the row's codes are formed with
struct RowScale {
  float s;    // int8: reciprocal of the row's scale; nvfp4: g
  float i6g;  // nvfp4: 1 / (6 g)
  bool bad;   // a value of the row is not finite: codes 0
};

// The block scale of a chunk with largest magnitude m (bits): its byte, and what
// the codes are multiplied with
template <int FMT>
__device__ __forceinline__ void block_scale(unsigned m, const RowScale& rs, uint32_t& byte, float& inv, bool& bad) {
  if (FMT == IC_MXFP4) {
    bad = m >= INF_BITS;
    const uint32_t e = m >> 23;
    byte = bad ? 255u : (e > 2 ? e - 2 : 0u);
    inv = __uint_as_float((254u - byte) << 23);  // bad: a subnormal, unused
  } else {
    bad = m >= INF_BITS || rs.bad;
    byte = bad ? (rs.bad ? 0u : 0x7fu) : to_e4m3(__fmul_rn(__uint_as_float(m), rs.i6g));
    inv = bad || byte == 0 ? 0.f : __frcp_rn(__fmul_rn(from_e4m3(byte), rs.s));
  }
}

// codes of one chunk of scaled values, and the scale bytes of four blocks as one word
template <int FMT>
__device__ __forceinline__ void store_fp4(const RowArgs& a, int64_t row, int64_t c, int64_t nch, const float (&y)[16],
                                          uint32_t byte, bool bad) {
  const int lane = threadIdx.x & 31;
  const uint32_t keep = bad ? 0u : 0xffffffffu;
  const uint2 codes = make_uint2(e2m1x8(y) & keep, e2m1x8(y + 8) & keep);
  const bool in = row < a.M && c < nch;
  if (in) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.q) + row * a.ldq + c * 8) = codes;
  // beyond the matrix the norm's 0 times its factor is NaN where that is not finite (a bad row, eps = 0): the bytes
  // there are zero (nvfp4: they are, such a row is bad)
  if (FMT == IC_MXFP4) byte = in ? byte : 0u;
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
}

// Codes of a pair of chunks (ca, cb) with largest magnitudes ma, mb; returns the sum of the int8 codes
template <int FMT>
__device__ __forceinline__ int emit_pair(const RowArgs& a, int64_t row, int64_t ca, int64_t cb, int64_t nch, f2 (&v)[16],
                                         unsigned ma, unsigned mb, const RowScale& rs) {
  float ya[16], yb[16];
  if (FMT == IC_INT8) {
    const f2 s = pk2(rs.s, rs.s);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const f2 y = mul2(v[j], s);
      ya[j] = lo2(y), yb[j] = hi2(y);
    }
    int sum = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float* y = h ? yb : ya;
      const int64_t c = h ? cb : ca;
      uint32_t w[4];
      int part = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        w[i] = rs.bad ? 0u : int8x4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
        part = __dp4a((int)w[i], 0x01010101, part);
      }
      if (row < a.M && c < nch) {
        *reinterpret_cast<uint4*>(static_cast<int8_t*>(a.q) + row * a.ldq + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
        sum += part;
      }
    }
    return sum;
  }
  if (FMT == IC_MXFP4) {  // a block is this chunk and the neighbouring lane's
    ma = max(ma, __shfl_xor_sync(0xffffffffu, ma, 1));
    mb = max(mb, __shfl_xor_sync(0xffffffffu, mb, 1));
  }
  uint32_t ba, bb;
  float ia, ib;
  bool xa, xb;
  block_scale<FMT>(ma, rs, ba, ia, xa);
  block_scale<FMT>(mb, rs, bb, ib, xb);
  const f2 inv = pk2(ia, ib);
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const f2 y = mul2(v[j], inv);
    ya[j] = lo2(y), yb[j] = hi2(y);
  }
  store_fp4<FMT>(a, row, ca, nch, ya, ba, xa);
  store_fp4<FMT>(a, row, cb, nch, yb, bb, xb);
  return 0;
}

// 16 elements as loaded, converted when they are used: loads stay ahead of the
// stores and reductions between them
template <typename T>
struct Raw {
  static constexpr int V = 16 / sizeof(T);
  uint4 r[16 / V];
  // elements at or beyond `left` are zero
  __device__ __forceinline__ void load(const T* p, int64_t left) {
    if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
      for (int i = 0; i < 16 / V; i += 2) load32(p + i * V, r[i], r[i + 1]);
    } else if (left >= 16 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
      for (int i = 0; i < 16 / V; ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16 / V; ++i) {
        T e[V];
#pragma unroll
        for (int u = 0; u < V; ++u) e[u] = i * V + u < left ? p[i * V + u] : from_f32<T>(0.f);
        r[i] = *reinterpret_cast<const uint4*>(e);
      }
    }
  }
  __device__ __forceinline__ float get(int j) const { return load_as_f32(reinterpret_cast<const T*>(&r[j / V]) + j % V); }
};

// the loads of a pair of chunks of one row
template <typename T, bool NORM>
struct RawPair {
  Raw<T> x[2], r[2];
  __device__ __forceinline__ void load(const RowArgs& a, int64_t row, int64_t ca, int64_t cb) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t c = h ? cb : ca, left = row < a.M ? a.K - c * 16 : 0;
      x[h].load(static_cast<const T*>(a.x) + (left > 0 ? row * a.ldx + c * 16 : 0), left);
      if (NORM && a.residual) r[h].load(static_cast<const T*>(a.residual) + (left > 0 ? row * a.ldr + c * 16 : 0), left);
    }
  }
  // h = x + residual as pairs, optionally written to residual_out
  __device__ __forceinline__ void add(const RowArgs& a, int64_t row, int64_t ca, int64_t cb, f2 (&v)[16], bool write) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = pk2(x[0].get(j), x[1].get(j));
    if (NORM && a.residual) {
#pragma unroll
      for (int j = 0; j < 16; ++j) v[j] = add2(v[j], pk2(r[0].get(j), r[1].get(j)));
      // the stream's value is rounded to its type here; the norm goes on from the sum in 32 bits
      if (write && row < a.M) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t c = h ? cb : ca;
          float y[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) y[j] = h ? hi2(v[j]) : lo2(v[j]);
          if (a.K > c * 16) store16(static_cast<T*>(a.residual_out) + row * a.ldo + c * 16, a.K - c * 16, y);
        }
      }
    }
  }
};
template <typename T, bool NORM>
__device__ __forceinline__ void load_pair(const RowArgs& a, int64_t row, int64_t ca, int64_t cb, f2 (&v)[16], bool write) {
  RawPair<T, NORM> p;
  p.load(a, row, ca, cb);
  p.add(a, row, ca, cb, v, write);
}

// (loading the weights ahead of the reduction as well took 126 instead of 80 registers and 47 instead of 39 us
// for 4608 x 4096 int8)
__device__ __forceinline__ void weigh_pair(const RowArgs& a, int64_t ca, int64_t cb, f2 (&v)[16], float rstd) {
  float x[16], y[16];
  load16_any(a.weight, a.wdtype, a.K - ca * 16 > 0 ? ca * 16 : 0, a.K - ca * 16, x);
  load16_any(a.weight, a.wdtype, a.K - cb * 16 > 0 ? cb * 16 : 0, a.K - cb * 16, y);
  const f2 r = pk2(rstd, rstd);
  // the last product is a scalar one: ptxas merges a packed product with the rotation's additions into
  // fused multiply-adds, which round differently from the product alone
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    const f2 h = mul2(v[j], r);
    v[j] = pk2(__fmul_rn(lo2(h), x[j]), __fmul_rn(hi2(h), y[j]));
  }
}

template <bool T256>
__device__ __forceinline__ void rotate_pair(const RowArgs& a, f2 (&v)[16], unsigned char* team) {
  if (T256) hadamard256(v, team, threadIdx.x & 15);
  else if (a.rot) hadamard_pair(v, a.rot, threadIdx.x & (a.rot / 16 - 1));
}
__device__ __forceinline__ void amax_pair(const f2 (&v)[16], unsigned& ma, unsigned& mb) {
  float x[16], y[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) x[j] = lo2(v[j]), y[j] = hi2(v[j]);
  ma = amax16(x);
  mb = amax16(y);
}

// A CTA takes groups of rows by turns and loads the next group's while it works
// on this one's (NP > 0): about a third of a row's time is otherwise spent
// waiting for HBM between two barriers.
template <typename T, int FMT, bool NORM, int NP, bool T256>
__global__ void __launch_bounds__(NP == 2 ? 512 : 256) rows_kernel(const RowArgs a) {
  __shared__ double buf[32];
  extern __shared__ __align__(16) unsigned char teams[];  // T256: TEAM_BYTES for every 16 threads
  unsigned char* team = teams + (threadIdx.x >> 4) * TEAM_BYTES;
  const int tpr = a.tpr, t = threadIdx.x & a.tmask, rpc = blockDim.x / tpr;
  const int64_t nch = cdiv(a.kp, 16);
  const int n = NP ? NP : (int)cdiv(nch, 2 * tpr);
  constexpr bool ROW = FMT != IC_MXFP4;  // the codes need the row's largest magnitude
  constexpr int R = NP ? NP : 1;
  auto ca = [&](int i) { return (int64_t)(2 * i) * tpr + t; };
  auto cb = [&](int i) { return (int64_t)(2 * i + 1) * tpr + t; };
  RawPair<T, NORM> raw[R];
  int64_t row = (int64_t)blockIdx.x * rpc + (threadIdx.x >> a.tshift);
  if (NP) {
#pragma unroll
    for (int i = 0; i < R; ++i) raw[i].load(a, row, ca(i), cb(i));
  }
  for (int64_t group = blockIdx.x; group < a.groups; group += gridDim.x, row += (int64_t)gridDim.x * rpc) {
    f2 v[R][16];
    unsigned ma[R], mb[R];
    float rstd = 0.f;
    if (NP) {
#pragma unroll
      for (int i = 0; i < R; ++i) raw[i].add(a, row, ca(i), cb(i), v[i], true);
      if (group + gridDim.x < a.groups) {
#pragma unroll
        for (int i = 0; i < R; ++i) raw[i].load(a, row + (int64_t)gridDim.x * rpc, ca(i), cb(i));
      }
    }
    auto finish = [&](int i, int k) {
      if (NORM) weigh_pair(a, ca(i), cb(i), v[k], rstd);
      rotate_pair<T256>(a, v[k], team);
      amax_pair(v[k], ma[k], mb[k]);
    };
    if (NORM) {
      double ss = 0.0;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        if (!NP) load_pair<T, NORM>(a, row, ca(i), cb(i), v[0], true);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const double x = lo2(v[NP ? i : 0][j]), y = hi2(v[NP ? i : 0][j]);
          ss = fma(x, x, ss);
          ss = fma(y, y, ss);
        }
      }
      ss = row_reduce(ss, tpr, a.tmask, buf, [](double p, double q) { return p + q; });
      // squares of fp32 values cannot overflow here: an infinite sum is an infinite input, which marks the whole row
      rstd = isfinite(ss) ? (float)(1.0 / sqrt(ss / (double)a.K + (double)a.eps)) : __int_as_float(0x7fc00000);
    }
    RowScale rs{0.f, 0.f, false};
    unsigned m = 0;
    if (NP || (ROW && !a.row_scale_in)) {
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const int k = NP ? i : 0;
        if (!NP) load_pair<T, NORM>(a, row, ca(i), cb(i), v[k], false);
        finish(i, k);
        m = max(m, max(ma[k], mb[k]));
      }
    }
    if (ROW) {
      float s;
      if (!a.row_scale_in) {
        m = __reduce_max_sync(0xffffffffu, m);
        m = row_reduce(m, tpr, a.tmask, reinterpret_cast<unsigned*>(buf), [](unsigned p, unsigned q) { return max(p, q); });
      }
      if (FMT == IC_INT8) {
        rs.bad = m >= INF_BITS;
        s = fmaxf(__fmul_rn(__uint_as_float(m), (float)(1.0 / 127.0)), LOWP_SCALE_FLOOR);
        rs.s = __frcp_rn(s);
      } else {
        if (a.row_scale_in) {
          s = row < a.M ? a.row_scale_in[row * a.rs_stride] : 1.f;
          rs.bad = !(s > 0.f) || __float_as_uint(s) >= INF_BITS;
          // it may be of any size: 1/(scale g) must not be infinite (0 * inf would make codes of zeros), nor 6 g
          rs.s = fmaxf(s, 0x1p-118f);
          const float far = s > 0x1p120f ? 0x1p-8f : 1.f;
          rs.i6g = __fmul_rn(__frcp_rn(__fmul_rn(6.f, __fmul_rn(rs.s, far))), far);
        } else {
          rs.bad = m >= INF_BITS;
          s = fmaxf(__fmul_rn(__uint_as_float(m), (float)(1.0 / 2688.0)), LOWP_SCALE_FLOOR);
          rs.s = s;
          rs.i6g = __frcp_rn(__fmul_rn(6.f, s));
        }
      }
      if (t == 0 && row < a.M) a.row_scale[row] = rs.bad ? __uint_as_float(0x7fc00000u) : s;
    }
    int sum = 0;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const int k = NP ? i : 0;
      if (!NP) {
        load_pair<T, NORM>(a, row, ca(i), cb(i), v[k], false);
        finish(i, k);
      }
      sum += emit_pair<FMT>(a, row, ca(i), cb(i), nch, v[k], ma[k], mb[k], rs);
    }
    if (FMT == IC_INT8 && a.sums) {
      sum = row_reduce(sum, tpr, a.tmask, reinterpret_cast<int*>(buf), [](int p, int q) { return p + q; });
      if (t == 0 && row < a.M) a.sums[row] = sum;
    }
  }
}

template <typename T, int FMT, bool NORM, int NP, bool T256>
int launch_np(const RowArgs& a, int threads, cudaStream_t st) {
  const auto kernel = rows_kernel<T, FMT, NORM, NP, T256>;
  const int smem = T256 ? threads / 16 * TEAM_BYTES : 0;
  // CTAs that the device holds at once, by device and warps of a block
  static std::atomic<int> resident[64][17];
  int dev = 0;
  IC_CUDA(cudaGetDevice(&dev));
  std::atomic<int>& r = resident[dev & 63][threads / 32];
  int ctas = r.load();
  if (!ctas) {
    int sms = 0;
    if (T256) IC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 32 * TEAM_BYTES));
    IC_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, threads, smem));
    IC_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    ctas = std::max(1, ctas) * sms;
    r.store(ctas);
  }
  const int64_t grid = NP ? std::min<int64_t>(a.groups, ctas) : a.groups;
  kernel<<<(unsigned)grid, threads, smem, st>>>(a);
  IC_CHECK_LAUNCH();
  return IC_OK;
}

template <typename T, int FMT, bool NORM>
int launch_rows(RowArgs a, cudaStream_t st) {
  const int64_t pairs = cdiv(cdiv(a.kp, 16), 2);
  // short rows: a power of two of threads, several rows to a CTA; then one row to a CTA with as many
  // warps as one pair of chunks per thread takes (two pairs beyond 256 threads), up to 512 threads
  int tpr = 32, np = 1;
  if (pairs <= 128) {
    while (tpr < pairs) tpr *= 2;
  } else {
    np = pairs <= 256 ? 1 : 2;
    tpr = (int)std::min<int64_t>(cdiv(cdiv(pairs, np), 32) * 32, 512);
    if ((int64_t)np * tpr < pairs) np = 0, tpr = 256;  // read again for each reduction
  }
  a.tpr = tpr;
  const int threads = std::max(tpr, 128);
  a.tshift = threads == tpr ? 10 : ilog2(tpr);
  a.tmask = (1 << a.tshift) - 1;
  // the 4-bit formats' scale tiles hold 128 rows: the grid covers the padding rows too
  const int64_t rows = FMT == IC_INT8 ? a.M : cdiv(a.M, 128) * 128;
  a.groups = cdiv(rows, threads / tpr);
  if (a.groups > INT32_MAX) return fail(IC_ERR_UNSUPPORTED, "quantize: too many rows");
  const bool t256 = a.rot == 256;
  if (np == 1) return t256 ? launch_np<T, FMT, NORM, 1, true>(a, threads, st) : launch_np<T, FMT, NORM, 1, false>(a, threads, st);
  if (np == 2) return t256 ? launch_np<T, FMT, NORM, 2, true>(a, threads, st) : launch_np<T, FMT, NORM, 2, false>(a, threads, st);
  return t256 ? launch_np<T, FMT, NORM, 0, true>(a, threads, st) : launch_np<T, FMT, NORM, 0, false>(a, threads, st);
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
// One chunk per thread; blockDim = (chunks of a row, rows), both powers of two.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) dequant_kernel(const uint8_t* __restrict__ q, int64_t ldq, int64_t M, int64_t kp,
                                                      const uint8_t* __restrict__ scales, int64_t ktiles,
                                                      const float* __restrict__ row_scale, T* __restrict__ out,
                                                      int64_t ldo) {
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y, left = kp - (int64_t)c * 16;
  if (row >= M || left <= 0) return;
  float v[16];
  if (FMT == IC_INT8) {
    const float s = row_scale[row];
    const int8_t* p = reinterpret_cast<const int8_t*>(q) + row * ldq + c * 16;
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
    const int b = FMT == IC_MXFP4 ? c >> 1 : c;
    const uint32_t byte = scales[scale_word(row, b >> 2, ktiles) + (b & 3)];
    const float s = FMT == IC_MXFP4 ? (byte == 255u ? __uint_as_float(0x7fc00000u)
                                                    : __uint_as_float(byte ? byte << 23 : 0x00400000u))
                                    : from_e4m3(byte);
    const float g = FMT == IC_NVFP4 ? row_scale[row] : 1.f;
    const uint2 raw = *reinterpret_cast<const uint2*>(q + row * ldq + (int64_t)c * 8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t h[4];  // two codes each as a pair of halves, exactly
      asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n"
          " cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n"
          " cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
          : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
          : "r"(i ? raw.y : raw.x));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
        f2 y = mul2(pk2(x.x, x.y), pk2(s, s));
        if (FMT == IC_NVFP4) y = mul2(y, pk2(g, g));
        v[i * 8 + j * 2] = lo2(y);
        v[i * 8 + j * 2 + 1] = hi2(y);
      }
    }
  }
  store16(out + row * ldo + (int64_t)c * 16, left, v);
}

template <int FMT>
int launch_dequant(const void* q, int64_t ldq, int64_t M, int64_t kp, const uint8_t* scales, int64_t ktiles,
                   const float* row_scale, int dtype, void* out, int64_t ldo, cudaStream_t st) {
  const uint8_t* p = static_cast<const uint8_t*>(q);
  const int64_t nch = cdiv(kp, 16);
  int tx = 1;
  while (tx < 256 && tx < nch) tx *= 2;
  const dim3 block(tx, 256 / tx);
  if (cdiv(nch, tx) > 65535 || cdiv(M, block.y) > INT32_MAX) return fail(IC_ERR_UNSUPPORTED, "dequantize: size");
  const dim3 grid((unsigned)cdiv(M, block.y), (unsigned)cdiv(nch, tx));
  switch (dtype) {
    case IC_F32: dequant_kernel<float, FMT><<<grid, block, 0, st>>>(p, ldq, M, kp, scales, ktiles, row_scale, (float*)out, ldo); break;
    case IC_F16: dequant_kernel<__half, FMT><<<grid, block, 0, st>>>(p, ldq, M, kp, scales, ktiles, row_scale, (__half*)out, ldo); break;
    case IC_BF16: dequant_kernel<__nv_bfloat16, FMT><<<grid, block, 0, st>>>(p, ldq, M, kp, scales, ktiles, row_scale, (__nv_bfloat16*)out, ldo); break;
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
