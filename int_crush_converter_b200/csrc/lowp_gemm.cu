// Products of low-precision operands on the 5th-generation tensor cores.
//
//   matmul_fp4:   y = (sum_blocks sa*sb * sum_k a*b) * ga * gb + bias   (E2M1 codes; mxfp4 or nvfp4 scales)
//   matmul_int8:  y = (sum_k a*w - zp * sum_k a) * sa * sw + bias        (exact int32 sums)
//
// One CTA computes a 128 x BN tile of the product of its "row" operand P
// (128 rows) and its "column" operand Q (BN rows), both K-major, 128 bytes of
// K per stage.  With many rows of activations P = activations; with few
// (`swap`) P = weights, so that 128 rows of tensor-core work are weight rows
// and the few activation rows set BN.  Warp roles (256 threads): warp 0 TMA
// producer, warp 1 MMA issuer, warp 2 TMEM allocator, warps 4-7 epilogue.
// The 4-bit kinds take their block scales from tensor memory: each stage's
// scale tiles come by bulk copy, and tcgen05.cp puts them in a ring of TMEM
// columns as deep as the stage ring, so a slot is rewritten only after the
// products that read it have finished.
//
// With few tiles a cluster of S CTAs splits K; each leaves its partial tile in
// its own shared memory and the cluster adds them in rank order, so the result
// does not depend on timing.  All waits are bounded (see common.cuh); where one
// gives up, the elements of y that it leaves without their sums are NaN.
//
// Measured on B200 (cuBLAS bf16 1700 TFLOP/s, copy 6.56 TB/s), launches in a
// graph: one row x 12288 x 4096 mxfp4 9.3 us with the weights in HBM, 7.9 us from
// L2 (25 MB: 4.1 us; a launch and its ends alone take 4.2 us); 512 x 4096 x 4096
// mxfp4 9.5 us, 300 x 4096 x 16384 nvfp4 20 us (bound by what L2 delivers to
// narrow tiles); large products run on CTA pairs, below.
#include <cstdlib>

#include "internal.h"
#include "lowp.cuh"

namespace ic {
namespace {

constexpr int BM = 128;
constexpr int ROW_BYTES = 128;  // K bytes per stage: one 128-byte swizzle row
constexpr unsigned WAIT_LIMIT_NS = 2000000000u;
constexpr int MAX_SPLIT = 8;

struct LowpArgs {
  int pm, qn;        // rows of P and Q
  int kbytes;        // bytes of K
  int ktiles;        // scale tiles (4 blocks) along K
  int splits;        // CTAs per tile (cluster size)
  int swap;          // P = weights: the output is transposed on the way out
  const uint8_t* p_scales;
  const uint8_t* q_scales;
  const void* p_row;  // per-row factors: fp32, or fp16 for INT8 weights; null: 1
  const void* q_row;
  int p_half, q_half;  // the factors are fp16
  const int8_t* zp;    // INT8 zero-points of the weights, or null
  const int32_t* sums; // row sums of the activations
  const void* bias;    // per weight row
  int bias_type;
  unsigned wait_ns;    // after which a wait gives up
  void* y;
  long long ldy;
  int out_type;
  int loads;           // stages that each CTA loads at most (the self-test of waits that give up)
  unsigned* flags;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const LowpArgs& a) {
  return mbar_wait_bounded(bar, parity, a.flags, a.wait_ns);
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// One lane of a converged warp.  The issuing warps run their loops with all
// lanes and elect around the instruction: addresses and descriptors then stay
// in uniform registers (a loop entered by one lane moved each operand of each
// instruction there, 67 cycles per tcgen05 instruction on B200).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
// every lane waits; true where all of them saw the phase complete (the warp stays converged either way)
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const LowpArgs& a) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, a));
}
// K-major operand in 128-byte swizzled rows: 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// one scale tile, 32 rows of 16 bytes without swizzle: 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)8 << 16 | (uint64_t)8 << 32 | (uint64_t)1 << 46;
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int KIND>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                    uint32_t accumulate) {
  if (KIND == IC_INT8)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else if (KIND == IC_MXFP4)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t saddr, uint32_t rank) {
  uint32_t out;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(out) : "r"(saddr), "r"(rank));
  return out;
}
__device__ __forceinline__ uint32_t ld_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// 16 accumulator columns of this warp's 32 lanes
#define IC_TMEM_LD16(taddr, r)                                                                                   \
  asm volatile(                                                                                                  \
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"   \
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),          \
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])     \
      : "r"(taddr))

#define IC_TMEM_LD32(taddr, r)                                                                   \
  asm volatile(                                                                                  \
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"   \
      "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"         \
      : "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]),      \
        "=r"((r)[6]), "=r"((r)[7]), "=r"((r)[8]), "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]),    \
        "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]), "=r"((r)[15]), "=r"((r)[16]), "=r"((r)[17]), \
        "=r"((r)[18]), "=r"((r)[19]), "=r"((r)[20]), "=r"((r)[21]), "=r"((r)[22]), "=r"((r)[23]), \
        "=r"((r)[24]), "=r"((r)[25]), "=r"((r)[26]), "=r"((r)[27]), "=r"((r)[28]), "=r"((r)[29]), \
        "=r"((r)[30]), "=r"((r)[31])                                                             \
      : "r"(taddr))

// What the epilogue applies to a 128 x BN tile: one side of it belongs to the
// activations (factor, sum of codes), the other to the weights (factor, bias,
// zero-point).
struct alignas(16) TileFactors {
  float rowf[128], rowb[128], colf[256], colb[256];
  int rowi[128], coli[256];
};

template <int KIND, int BN>
struct Cfg {
  static constexpr bool FP4 = KIND != IC_INT8;
  static constexpr int SF_TILES = KIND == IC_NVFP4 ? 4 : KIND == IC_MXFP4 ? 2 : 0;  // scale tiles per stage and 128 rows
  static constexpr int Q_ATOMS = BN > 128 ? 2 : 1;
  static constexpr int P_BYTES = BM * ROW_BYTES;
  static constexpr int Q_BYTES = BN * ROW_BYTES;
  static constexpr int PS_BYTES = SF_TILES * 512;
  static constexpr int QS_BYTES = SF_TILES * 512 * Q_ATOMS;
  static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES + PS_BYTES + QS_BYTES;
  // narrow tiles leave room for two CTAs on an SM; wide ones take the SM
  static constexpr int CTAS = BN <= 64 ? 2 : 1;
  static constexpr int STAGES = (CTAS == 2 ? 98304 : 222000) / STAGE_BYTES;
  static constexpr int SF_COLS = SF_TILES * 4 * (1 + Q_ATOMS);  // TMEM columns of one stage's scales
  static constexpr int ACC_COLS = BN < 32 ? 32 : BN;
  static constexpr int TMEM_NEED = ACC_COLS + STAGES * SF_COLS;
  static constexpr int TMEM_COLS = TMEM_NEED <= 32 ? 32 : TMEM_NEED <= 64 ? 64 : TMEM_NEED <= 128 ? 128 : TMEM_NEED <= 256 ? 256 : 512;
  static constexpr int SMEM = STAGES * STAGE_BYTES + (int)sizeof(TileFactors) + 1024 /*align*/ + 256 /*barriers*/;
  static_assert(TMEM_NEED <= 512 / CTAS, "tensor memory");
  static_assert(STAGE_BYTES % 1024 == 0 && sizeof(TileFactors) % 16 == 0, "stages in whole swizzle patterns, barriers on 8 bytes");
  static_assert(8 * (2 * STAGES + 2) + 4 <= 256, "barriers");
  static_assert(SMEM <= 232448 / CTAS, "shared memory");
  static_assert(BM * BN * 4 <= STAGES * STAGE_BYTES, "a partial tile fits in the stages");
  static constexpr uint32_t IDESC =
      KIND == IC_INT8 ? (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24)
                      : (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (KIND == IC_MXFP4 ? 1u << 23 : 0u) |
                            ((uint32_t)(BM >> 4) << 24);
};

__device__ __forceinline__ float load_any(const void* p, int type, long long i) {
  if (type == IC_F32) return static_cast<const float*>(p)[i];
  if (type == IC_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
// v[i] = p[first + 32 i], zero beyond `limit` or without p; the loads of all N are in flight together
template <int N>
__device__ __forceinline__ void load_strided(const void* p, int type, int first, int limit, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = 0.f;
  if (!p) return;
  if (type == IC_F32) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first + 32 * i < limit) v[i] = static_cast<const float*>(p)[first + 32 * i];
  } else if (type == IC_F16) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first + 32 * i < limit) v[i] = __half2float(static_cast<const __half*>(p)[first + 32 * i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first + 32 * i < limit) v[i] = __bfloat162float(static_cast<const __nv_bfloat16*>(p)[first + 32 * i]);
  }
}
// One sum to its output: fp32 scaling in a fixed order (zero-point, the
// activations' factor, the weights' factor, bias), rounded to the output type
// once, by the caller.
template <int KIND>
__device__ __forceinline__ float finish(uint32_t acc, int zs, float tokf, float wf, float bias, bool has_bias) {
  float v = KIND == IC_INT8 ? (float)((int)acc - zs) : __uint_as_float(acc);
  if (KIND != IC_MXFP4) v = __fmul_rn(__fmul_rn(v, tokf), wf);
  return has_bias ? __fadd_rn(v, bias) : v;
}
template <typename T>
__device__ __forceinline__ T to_out(float v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(v);
  else return __float2bfloat16_rn(v);
}
// Where a wait gave up the sums are not there: NaN, so that no caller takes what lies in y for a product.
// `rows` x `cols` elements of y from element `at`, the lanes side by side along its rows.
__device__ __forceinline__ void store_nan(const LowpArgs& a, long long at, int rows, int cols, int lane) {
#pragma unroll 1
  for (int r = 0; r < rows; ++r, at += a.ldy)
#pragma unroll 1
    for (int c = lane; c < cols; c += 32) {
      if (a.out_type == IC_F32) static_cast<uint32_t*>(a.y)[at + c] = 0x7fffffffu;
      else static_cast<uint16_t*>(a.y)[at + c] = 0x7fffu;  // in both 16-bit types
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* to, const T (&e)[V]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(e);
  if constexpr (V * sizeof(T) == 32)
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                 "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
  else
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(e);
}

// A warp's 32 rows of C columns through its shared memory `mine` (68 bytes a
// row: the banks stay apart) to rows of y that are not 16-byte aligned:
// neighbouring lanes store neighbouring elements.  v: this lane's row.
constexpr int ROW_PITCH = 68;
template <typename T, int C>
__device__ __forceinline__ void store_rows(unsigned char* mine, const float (&v)[C], int rows, int cols, T* to, long long ld,
                                           int lane) {
  static_assert(C * sizeof(T) <= 64 && 32 % C == 0, "a row of the buffer");
  uint32_t* w = reinterpret_cast<uint32_t*>(mine + lane * ROW_PITCH);
#pragma unroll
  for (int j = 0; j < C * (int)sizeof(T) / 4; ++j) {
    if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(v[j]);
    else {
      T e[2] = {to_out<T>(v[2 * j]), to_out<T>(v[2 * j + 1])};
      w[j] = *reinterpret_cast<const uint32_t*>(e);
    }
  }
  __syncwarp();
  constexpr int R = 32 / C;  // rows at a time
  const int i = lane % C;
#pragma unroll 8
  for (int k = 0; k < 32; k += R) {
    const int r = k + lane / C;
    const T x = reinterpret_cast<const T*>(mine + r * ROW_PITCH)[i];
    if (r < rows && i < cols) to[r * ld + i] = x;
  }
  __syncwarp();
}

// factors of a tile's rows and columns, by 128 threads
template <int BN>
__device__ __forceinline__ void load_factors(const LowpArgs& a, TileFactors& f, int p0, int q0, int t) {
  const int row = p0 + t;
  const bool in = row < a.pm;
  f.rowf[t] = in && a.p_row ? load_any(a.p_row, a.p_half ? IC_F16 : IC_F32, row) : 0.f;
  f.rowb[t] = in && a.swap && a.bias ? load_any(a.bias, a.bias_type, row) : 0.f;
  f.rowi[t] = in && a.zp ? (a.swap ? (int)a.zp[row] : a.sums[row]) : 0;
#pragma unroll
  for (int i = 0; i < (BN + 127) / 128; ++i) {
    const int c = i * 128 + t, col = q0 + c;
    if (c >= BN) break;
    const bool on = col < a.qn;
    f.colf[c] = on && a.q_row ? load_any(a.q_row, a.q_half ? IC_F16 : IC_F32, col) : 0.f;
    f.colb[c] = on && !a.swap && a.bias ? load_any(a.bias, a.bias_type, col) : 0.f;
    f.coli[c] = on && a.zp ? (a.swap ? a.sums[col] : (int)a.zp[col]) : 0;
  }
}

// In place of a partial sum where a wait gave up: NaN, or the integer that no sum of int8 products is (k < 2^17)
constexpr uint32_t NO_SUM = 0x80000000u;

// This CTA's share of a split tile's columns: the S partial sums in rank order, then to y
template <int KIND, int BN, int S, typename T>
__device__ __forceinline__ void add_parts(const LowpArgs& a, const TileFactors& f, T* y, const uint32_t* part, int p0, int q0,
                                          int rank) {
  constexpr int SHARE = BN / S, V = SHARE < 16 / (int)sizeof(T) ? SHARE : 16 / (int)sizeof(T);  // columns: in all, at a time
  const int lr = threadIdx.x & 127, row = p0 + lr, c0 = rank * SHARE, left = min(SHARE, a.qn - q0 - c0);
  uint32_t peer[S];
#pragma unroll
  for (int r = 0; r < S; ++r) peer[r] = map_to_rank(smem_u32(part + c0 * BM + lr), r);
  const float rowf = f.rowf[lr], rowb = f.rowb[lr];
  const int rowi = f.rowi[lr];
  const bool has_bias = a.bias != nullptr;
  const bool vec = !a.swap && V * sizeof(T) == 16 && ((reinterpret_cast<uintptr_t>(y) | (uintptr_t)(a.ldy * (long long)sizeof(T))) & 15) == 0;
  for (int g = (threadIdx.x >> 7) * V; g < left; g += 2 * V) {
    uint32_t v[V][S];  // all loads in flight together
#pragma unroll
    for (int u = 0; u < V; ++u)
#pragma unroll
      for (int r = 0; r < S; ++r) v[u][r] = ld_cluster(peer[r] + (uint32_t)((g + u) * BM) * 4u);
    alignas(16) T e[V];
#pragma unroll
    for (int u = 0; u < V; ++u) {
      const int c = c0 + g + u;
      uint32_t s = v[u][0];
      bool bad = KIND == IC_INT8 && s == NO_SUM;
#pragma unroll
      for (int r = 1; r < S; ++r) {
        if (KIND == IC_INT8) s += v[u][r], bad |= v[u][r] == NO_SUM;
        else s = __float_as_uint(__fadd_rn(__uint_as_float(s), __uint_as_float(v[u][r])));
      }
      const float cf = f.colf[c];
      const float x = finish<KIND>(s, rowi * f.coli[c], a.swap ? cf : rowf, a.swap ? rowf : cf, a.swap ? rowb : f.colb[c], has_bias);
      e[u] = to_out<T>(bad ? __uint_as_float(0x7fffffffu) : x);
    }
    if (row >= a.pm) continue;
    const int col = q0 + c0 + g;
    if (a.swap) {
#pragma unroll
      for (int u = 0; u < V; ++u)
        if (g + u < left) y[(long long)(col + u) * a.ldy + row] = e[u];
    } else if (vec && g + V <= left && col % V == 0) {
      if constexpr (V * sizeof(T) == 16) store_vec<T, V>(y + (long long)row * a.ldy + col, e);
    } else {
#pragma unroll
      for (int u = 0; u < V; ++u)
        if (g + u < left) y[(long long)row * a.ldy + col + u] = e[u];
    }
  }
}

// Sums to y.  The accumulator's lanes are rows of P, its columns rows of Q.
//  - one CTA per tile, activations in P: each lane stores pieces of its own row
//    of y (whole sectors where the rows are aligned; otherwise through shared
//    memory, neighbouring lanes storing neighbouring elements);
//  - weights in P: lanes are neighbouring columns of y, stored as they are;
//  - split K: partial tiles go to shared memory as [column][128 rows], each CTA
//    of the cluster adds its share of the columns over the CTAs in rank order.
template <int KIND, int BN, typename T>
__device__ __forceinline__ void epilogue(const LowpArgs& a, const TileFactors& f, unsigned char* smem, uint32_t tmem,
                                         uint32_t acc_bar, int p0, int q0, int rank) {
  constexpr int W = BN < 32 ? 16 : 32;  // columns at a time
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3;
  T* y = static_cast<T*>(a.y);
  const bool has_bias = a.bias != nullptr;
  uint32_t* part = reinterpret_cast<uint32_t*>(smem);
  if (warp >= 4) {
    asm volatile("bar.sync 1, 128;" ::: "memory");  // the factors are written
    const bool ok = warp_wait(acc_bar, 0, a);
    asm volatile("tcgen05.fence::after_thread_sync;");
    const int lr = q * 32 + lane, row = p0 + lr;
    const float rowf = f.rowf[lr], rowb = f.rowb[lr];
    const int rowi = f.rowi[lr];
    constexpr int V = 32 / sizeof(T);
    const uintptr_t at_y = reinterpret_cast<uintptr_t>(y) | (uintptr_t)(a.ldy * (long long)sizeof(T));
    const bool vec = !a.swap && (at_y & 15) == 0, whole = (at_y & 31) == 0;
    const int cols = min(BN, a.qn - q0), rows = min(32, a.pm - p0 - q * 32);
    if (!ok && a.splits > 1) {
      for (int c = 0; c < cols; ++c) part[c * BM + lr] = KIND == IC_INT8 ? NO_SUM : 0x7fffffffu;
    } else if (!ok) {
      if (a.swap) store_nan(a, (long long)q0 * a.ldy + p0 + q * 32, cols, rows, lane);
      else store_nan(a, (long long)(p0 + q * 32) * a.ldy + q0, rows, cols, lane);
    }
    for (int c = 0; ok && c < cols; c += W) {
      uint32_t r[W];
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)c;
      if constexpr (W == 16) IC_TMEM_LD16(at, r);
      else IC_TMEM_LD32(at, r);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (a.splits > 1) {
#pragma unroll
        for (int j = 0; j < W; ++j) part[(c + j) * BM + lr] = r[j];
        continue;
      }
      float v[W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float cf = f.colf[c + j];
        v[j] = finish<KIND>(r[j], rowi * f.coli[c + j], a.swap ? cf : rowf, a.swap ? rowf : cf, a.swap ? rowb : f.colb[c + j], has_bias);
      }
      if (a.swap) {
        if (row < a.pm) {
          T* to = y + (long long)(q0 + c) * a.ldy + row;
#pragma unroll
          for (int j = 0; j < W; ++j)
            if (c + j < cols) to[j * a.ldy] = to_out<T>(v[j]);
        }
      } else if (vec) {
        T* to = y + (long long)row * a.ldy + q0 + c;
        const int left = row < a.pm ? cols - c : 0;
#pragma unroll
        for (int j = 0; j < W; j += V) {
          alignas(32) T e[V];
#pragma unroll
          for (int u = 0; u < V; ++u) e[u] = to_out<T>(v[j + u]);
          if (j + V <= left && whole) {
            store_vec<T, V>(to + j, e);
          } else if (j + V <= left) {
            *reinterpret_cast<uint4*>(to + j) = *reinterpret_cast<const uint4*>(e);
            *reinterpret_cast<uint4*>(to + j + V / 2) = *reinterpret_cast<const uint4*>(e + V / 2);
          } else
#pragma unroll
            for (int u = 0; u < V; ++u)
              if (j + u < left) to[j + u] = e[u];
        }
      } else {
        unsigned char* mine = smem + q * (32 * ROW_PITCH);  // the stages are idle by now
        constexpr int C = 64 / sizeof(T) < W ? 64 / sizeof(T) : W;
#pragma unroll
        for (int g = 0; g < W; g += C) {
          float part_v[C];
#pragma unroll
          for (int u = 0; u < C; ++u) part_v[u] = v[g + u];
          store_rows<T, C>(mine, part_v, rows, min(C, cols - c - g),
                           y + (long long)(p0 + q * 32) * a.ldy + q0 + c + g, a.ldy, lane);
        }
      }
    }
  }
  if (a.splits > 1) {
    cluster_sync();
    if (a.splits == 2) add_parts<KIND, BN, 2>(a, f, y, part, p0, q0, rank);
    else if (a.splits == 4) add_parts<KIND, BN, 4>(a, f, y, part, p0, q0, rank);
    else add_parts<KIND, BN, 8>(a, f, y, part, p0, q0, rank);
    cluster_sync();  // no CTA leaves while a peer reads its partial tile
  }
}

constexpr int GROUP = 16;  // row tiles per group of the tile order: a wave of CTAs reads a compact patch of P and Q

template <int KIND, int BN>
__global__ void __launch_bounds__(256, Cfg<KIND, BN>::CTAS)
    lowp_gemm_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ, const LowpArgs a) {
  using C = Cfg<KIND, BN>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  TileFactors& f = *reinterpret_cast<TileFactors*>(smem + STAGES * C::STAGE_BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGES * C::STAGE_BYTES + sizeof(TileFactors));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 2);
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + STAGES + s); };
  const uint32_t acc_bar = smem_u32(bars + 2 * STAGES), last_bar = smem_u32(bars + 2 * STAGES + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / a.splits, rank = blockIdx.x - tile * a.splits;
  const int pt = (a.pm + BM - 1) / BM, qt = (a.qn + BN - 1) / BN;
  const int per = GROUP * qt, grp = tile / per, first = grp * GROUP, gm = min(GROUP, pt - first), local = tile - grp * per;
  const int p0 = (first + local % gm) * BM, q0 = (local / gm) * BN;
  const int stages_all = (a.kbytes + ROW_BYTES - 1) / ROW_BYTES;
  const int kt0 = (int)((long long)rank * stages_all / a.splits), kt1 = (int)((long long)(rank + 1) * stages_all / a.splits);
  const int n = kt1 - kt0;  // at least one: the host splits no further than the stages

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    mbar_init(acc_bar, 1);
    mbar_init(last_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer ----------------
    int issued = 0;
    const int loads = min(n, a.loads);
    for (int i = 0; i < loads; ++i) {
      const int s = i % STAGES;
      if (i >= STAGES && !mbar_wait(empty_bar(s), ((i / STAGES) & 1) ^ 1, a)) break;
      const int kt = kt0 + i;
      const uint32_t base = smem_u32(smem + s * C::STAGE_BYTES);
      uint32_t bytes = C::P_BYTES + C::Q_BYTES, sf = 0;
      const int rt = q0 >> 7;
      const bool two = C::Q_ATOMS == 2 && (rt + 1) * BM < a.qn;
      if (C::FP4) {
        sf = (uint32_t)min(C::SF_TILES, a.ktiles - kt * C::SF_TILES) * 512u;  // at least one tile: kt is within K
        bytes += sf * (two ? 3u : 2u);
      }
      mbar_expect_tx(full_bar(s), bytes);
      tma_load_2d(base, &tmP, kt * ROW_BYTES, p0, full_bar(s));
      tma_load_2d(base + C::P_BYTES, &tmQ, kt * ROW_BYTES, q0, full_bar(s));
      if (C::FP4) {
        const uint32_t ps = base + C::P_BYTES + C::Q_BYTES, qs = ps + C::PS_BYTES;
        const long long k = (long long)kt * C::SF_TILES;
        bulk_load(ps, a.p_scales + ((long long)(p0 >> 7) * a.ktiles + k) * 512, sf, full_bar(s));
        bulk_load(qs, a.q_scales + ((long long)rt * a.ktiles + k) * 512, sf, full_bar(s));
        if (two) bulk_load(qs + C::PS_BYTES, a.q_scales + ((long long)(rt + 1) * a.ktiles + k) * 512, sf, full_bar(s));
      }
      issued = i + 1;
    }
    // no copy of this CTA is in flight when it leaves (already true unless a wait gave up)
    for (int i = max(0, issued - STAGES); i < issued; ++i)
      mbar_wait_bounded(full_bar(i % STAGES), (i / STAGES) & 1, a.flags, WAIT_LIMIT_NS);
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    const uint32_t base0 = smem_u32(smem), sf0 = tmem + C::ACC_COLS;
    const uint64_t pd = operand_desc(base0), qd = operand_desc(base0 + C::P_BYTES), sd = scale_desc(base0 + C::P_BYTES + C::Q_BYTES);
    const uint32_t qcol = C::FP4 ? (uint32_t)((q0 & 127) >> 5) : 0u;  // narrow tiles start inside a 128-row scale tile
    int s = 0, left = a.kbytes - kt0 * ROW_BYTES;
    uint32_t ph = 0;
    bool ok = true;
    for (int i = 0; i < n; ++i, left -= ROW_BYTES) {
      ok = warp_wait(full_bar(s), ph, a);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;");
      const uint32_t at = (uint32_t)(s * C::STAGE_BYTES) >> 4;  // the descriptors' address field counts 16 bytes
      const uint32_t sfp = sf0 + s * C::SF_COLS, sfq = sfp + C::SF_TILES * 4;
      const int steps = min(4, (left + 31) >> 5);  // 32 bytes of K each
      if (elect_one()) {
        if (C::FP4) {
          const int tiles = KIND == IC_NVFP4 ? steps : (steps + 1) / 2;
#pragma unroll
          for (int t = 0; t < C::SF_TILES; ++t) {
            if (t >= tiles) break;
            copy_scales(sfp + t * 4, sd + at + t * 32);
#pragma unroll
            for (int u = 0; u < C::Q_ATOMS; ++u)
              copy_scales(sfq + (t * C::Q_ATOMS + u) * 4, sd + at + ((u + 1) * C::PS_BYTES >> 4) + t * 32);
          }
        }
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          if (kk >= steps) break;
          const int t = KIND == IC_NVFP4 ? kk : kk >> 1;
          const uint32_t id = KIND == IC_MXFP4 && (kk & 1) ? C::IDESC | (2u << 4) | (2u << 29) : C::IDESC;
          mma<KIND>(tmem, pd + at + kk * 2, qd + at + kk * 2, id, sfp + t * 4, sfq + t * C::Q_ATOMS * 4 + qcol, (i | kk) ? 1u : 0u);
        }
        mma_commit(empty_bar(s));
        if (i == n - 1) mma_commit(acc_bar);
      }
      __syncwarp();
      if (++s == STAGES) {
        s = 0;
        ph ^= 1;
      }
    }
    // products in flight end before their tensor memory is freed
    if (!ok && elect_one()) mma_commit(last_bar);
    __syncwarp();
    mbar_wait_bounded(ok ? acc_bar : last_bar, 0, a.flags, WAIT_LIMIT_NS);
  }
  __syncwarp();

  // ---------------- epilogue ----------------
  if (warp >= 4) load_factors<BN>(a, f, p0, q0, threadIdx.x - 128);
  if (a.out_type == IC_BF16) epilogue<KIND, BN, __nv_bfloat16>(a, f, smem, tmem, acc_bar, p0, q0, rank);
  else if (a.out_type == IC_F16) epilogue<KIND, BN, __half>(a, f, smem, tmem, acc_bar, p0, q0, rank);
  else epilogue<KIND, BN, float>(a, f, smem, tmem, acc_bar, p0, q0, rank);
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
  }
}

// ---------------------------------------------------------------------------
// CTA pairs (cta_group::2) for large products: a cluster of two CTAs computes
// 256 x 256 tiles, one after another, each CTA staging its own 128 rows of P
// and of Q and the scales of its P rows and of all Q rows.  Per SM and 128
// bytes of K that is 32 KB of operands for 512 tensor-core cycles; a single
// CTA's 128 x 128 tile needs 32 KB for 256, more than L2 delivers.
// Tensor memory: INT8 has two accumulators of 256 columns, by turns.  The 4-bit
// kinds have one and every stage's scales (overlapping two accumulators left
// room for the scales of three stages: 127 instead of 117 us at
// 4608 x 4096 x 16384 nvfp4).  Eight epilogue warps move an accumulator to
// registers at once and release it; scaling, conversion and stores run under
// the next products.
//
// Measured on B200, a few calls at full clocks: 4608 x 16384 x 4096 nvfp4 134 us
// (4.6 PFLOP/s), 4608 x 4096 x 16384 nvfp4 111 us (5.6), 4608 x 12288 x 4096 int8
// 149 us (3.1 POP/s), 4608 x 4096 x 16384 int8 200 us (3.1); call after call under
// the power cap the first takes 168 us (3.7), the third 186 us (2.5).  In clocks
// the INT8 main loop runs at 530 a stage of 512, the nvfp4 one at 618: 38,912 bytes
// a stage at the 63 bytes a clock that L2 delivers to an SM.  About 3000 clocks are
// lost between two tiles of the 4-bit kinds' one accumulator.
//   full[s]  leader only: the bytes of both CTAs' loads
//   empty[s] in each CTA: the commit of the products that read the stage
//   accf[b]  in each CTA: the commit of a tile's last product into accumulator b
//   acce[b]  leader only: 16 epilogue warps have taken accumulator b
//   facf/face[b] in each CTA: the tile's factors are loaded / have been read
//   last     leader only: the commit of the products before a wait that gave up
// What the epilogue applies to one 128 x 256 part of a tile
struct Factors {
  float col[256], bias[256], row[128];
  int zp[256], sum[128];
};

constexpr int PAIR_GROUP = 8;  // 256-row tiles per group of the tile order

template <int KIND>
struct PairCfg {
  static constexpr bool FP4 = KIND != IC_INT8;
  static constexpr int BN = 256;
  static constexpr int SF_TILES = KIND == IC_NVFP4 ? 4 : KIND == IC_MXFP4 ? 2 : 0;
  static constexpr int P_BYTES = 128 * ROW_BYTES, Q_BYTES = 128 * ROW_BYTES;
  static constexpr int PS_BYTES = SF_TILES * 512, QS_BYTES = 2 * PS_BYTES;
  static constexpr int STAGE_BYTES = P_BYTES + Q_BYTES + PS_BYTES + QS_BYTES;
  static constexpr int STAGES = FP4 ? 5 : 6;
  static constexpr int SF_COLS = SF_TILES * 12;
  static constexpr int NACC = FP4 ? 1 : 2;
  static constexpr int TMEM_COLS = 512;
  static constexpr int OUT_BYTES = 8 * 32 * ROW_PITCH;  // per epilogue warp: 32 rows of 64 bytes
  static constexpr int SMEM = STAGES * STAGE_BYTES + OUT_BYTES + 2 * (int)sizeof(Factors) + 1024 + 256;
  static_assert(NACC * BN + STAGES * SF_COLS <= TMEM_COLS, "tensor memory");
  static_assert(STAGE_BYTES % 1024 == 0 && OUT_BYTES % 16 == 0 && sizeof(Factors) % 16 == 0, "stages in whole swizzle patterns, barriers on 8 bytes");
  static_assert(8 * (2 * STAGES + 9) + 4 <= 256, "barriers");
  static_assert(SMEM <= 232448, "shared memory");
  static constexpr uint32_t IDESC =
      KIND == IC_INT8 ? (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(256 >> 4) << 24)
                      : (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (KIND == IC_MXFP4 ? 1u << 23 : 0u) |
                            ((uint32_t)(256 >> 4) << 24);
};

__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
      "[%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int KIND>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                         uint32_t accumulate) {
  if (KIND == IC_INT8)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  else if (KIND == IC_MXFP4)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  const uint16_t mask = 3;
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask)
      : "memory");
}
__device__ __forceinline__ void mma_commit_leader(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void remote_arrive(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// One lane's row of four sums from column c of the tile, scaled
template <int KIND>
__device__ __forceinline__ void finish4(const LowpArgs& a, const uint32_t* acc, const Factors& f, int c, float rowf, int sum,
                                        float (&v)[4]) {
  float s[4] = {1.f, 1.f, 1.f, 1.f}, b[4];
  if (KIND != IC_MXFP4) *reinterpret_cast<float4*>(s) = *reinterpret_cast<const float4*>(f.col + c);
  if (a.bias) *reinterpret_cast<float4*>(b) = *reinterpret_cast<const float4*>(f.bias + c);
  int z[4];
  if (KIND == IC_INT8 && a.zp) *reinterpret_cast<int4*>(z) = *reinterpret_cast<const int4*>(f.zp + c);
#pragma unroll
  for (int u = 0; u < 4; ++u)
    v[u] = finish<KIND>(acc[u], KIND == IC_INT8 && a.zp ? z[u] * sum : 0, rowf, s[u], a.bias ? b[u] : 0.f, a.bias != nullptr);
}

// One warp's 32 rows x 128 columns of sums, from column c0 of the tile, to y.
// Rows that are 32-byte (16-byte) aligned: each lane stores its own row in whole
// (half) sectors, past shared memory, whose bandwidth the loads and products of the
// next tile take up.  Other rows: through the warp's part `out` of it, 64 bytes
// of each row at a time.
template <int KIND, typename T>
__device__ __forceinline__ void store_block(const LowpArgs& a, const uint32_t (&acc)[128], unsigned char* out,
                                            const Factors& f, int r0, int c0, int row0, int col0, int lane) {
  T* y = static_cast<T*>(a.y);
  const float rowf = f.row[r0 + lane];
  const int sum = f.sum[r0 + lane];
  const uintptr_t at = reinterpret_cast<uintptr_t>(y) | (uintptr_t)(a.ldy * (long long)sizeof(T));
  if ((at & 15) == 0) {
    constexpr int V = 32 / sizeof(T);
    const bool whole = (at & 31) == 0;
    T* to = y + (long long)(row0 + lane) * a.ldy + col0;
    const int left = row0 + lane < a.pm ? a.qn - col0 : 0;
#pragma unroll
    for (int c = 0; c < 128; c += V) {
      alignas(32) T e[V];
#pragma unroll
      for (int u = 0; u < V; u += 4) {
        float v[4];
        finish4<KIND>(a, acc + c + u, f, c0 + c + u, rowf, sum, v);
#pragma unroll
        for (int w = 0; w < 4; ++w) e[u + w] = to_out<T>(v[w]);
      }
      if (c + V <= left && whole) {
        store_vec<T, V>(to + c, e);
      } else if (c + V <= left) {
        *reinterpret_cast<uint4*>(to + c) = *reinterpret_cast<const uint4*>(e);
        *reinterpret_cast<uint4*>(to + c + V / 2) = *reinterpret_cast<const uint4*>(e + V / 2);
      } else {
#pragma unroll
        for (int u = 0; u < V; ++u)
          if (c + u < left) to[c + u] = e[u];
      }
    }
    return;
  }
  constexpr int G = 64 / sizeof(T);  // columns at a time
#pragma unroll
  for (int g = 0; g < 128; g += G) {
    float v[G];
#pragma unroll
    for (int u = 0; u < G; u += 4) {
      float x[4];
      finish4<KIND>(a, acc + g + u, f, c0 + g + u, rowf, sum, x);
#pragma unroll
      for (int w = 0; w < 4; ++w) v[u + w] = x[w];
    }
    store_rows<T, G>(out, v, min(32, a.pm - row0), min(G, a.qn - col0 - g), y + (long long)row0 * a.ldy + col0 + g, a.ldy, lane);
  }
}

template <int KIND>
__global__ void __launch_bounds__(384, 1)
    lowp_pair_kernel(const __grid_constant__ CUtensorMap tmP, const __grid_constant__ CUtensorMap tmQ,
                     const __grid_constant__ CUtensorMap tmPS, const __grid_constant__ CUtensorMap tmQS, const LowpArgs a) {
  using C = PairCfg<KIND>;
  constexpr int STAGES = C::STAGES;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* out_smem = smem + STAGES * C::STAGE_BYTES;
  Factors* factors = reinterpret_cast<Factors*>(out_smem + C::OUT_BYTES);  // two, by turns
  uint64_t* bars = reinterpret_cast<uint64_t*>(out_smem + C::OUT_BYTES + 2 * sizeof(Factors));
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 9);
  auto full_bar = [&](int s) { return smem_u32(bars + s); };
  auto empty_bar = [&](int s) { return smem_u32(bars + STAGES + s); };
  auto accf = [&](int b) { return smem_u32(bars + 2 * STAGES + b); };
  auto acce = [&](int b) { return smem_u32(bars + 2 * STAGES + 2 + b); };
  auto facf = [&](int b) { return smem_u32(bars + 2 * STAGES + 4 + b); };
  auto face = [&](int b) { return smem_u32(bars + 2 * STAGES + 6 + b); };
  const uint32_t last_bar = smem_u32(bars + 2 * STAGES + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  const int pt = (a.pm + 255) / 256, qt = (a.qn + C::BN - 1) / C::BN, tiles = pt * qt;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int n = (a.kbytes + ROW_BYTES - 1) / ROW_BYTES;
  auto place = [&](int tile, int& p0, int& q0) {
    const int per = PAIR_GROUP * qt, grp = tile / per, first = grp * PAIR_GROUP, gm = min(PAIR_GROUP, pt - first);
    const int local = tile - grp * per;
    p0 = (first + local % gm) * 256;
    q0 = (local / gm) * C::BN;
  };

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(accf(b), 1);
      mbar_init(acce(b), 16);
      mbar_init(facf(b), 32);
      mbar_init(face(b), 8);
    }
    mbar_init(last_bar, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(C::TMEM_COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;");
  const uint32_t tmem = *tmem_slot;

  if (warp == 0 && lane == 0) {
    // ---------------- TMA producer (both CTAs) ----------------
    int g = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      int p0, q0;
      place(tile, p0, q0);
      for (int i = 0; i < n; ++i, ++g) {
        const int s = g % STAGES;
        if (g >= a.loads || (g >= STAGES && !mbar_wait(empty_bar(s), ((g / STAGES) & 1) ^ 1, a))) {
          ok = false;
          break;
        }
        if (leader) mbar_expect_tx(full_bar(s), 2 * C::STAGE_BYTES);
        const uint32_t fb = map_to_rank(full_bar(s), 0);
        const uint32_t base = smem_u32(smem + s * C::STAGE_BYTES);
        tma_load_2d_pair(base, &tmP, i * ROW_BYTES, p0 + (int)rank * 128, fb);
        tma_load_2d_pair(base + C::P_BYTES, &tmQ, i * ROW_BYTES, q0 + (int)rank * 128, fb);
        if (C::FP4) {
          const uint32_t ps = base + C::P_BYTES + C::Q_BYTES;
          tma_load_3d_pair(ps, &tmPS, 0, i * C::SF_TILES, (p0 >> 7) + (int)rank, fb);
          tma_load_3d_pair(ps + C::PS_BYTES, &tmQS, 0, i * C::SF_TILES, q0 >> 7, fb);
        }
      }
    }
    // no copy is in flight when the pair leaves (already true unless a wait gave up)
    if (leader)
      for (int i = max(0, g - STAGES); i < g; ++i)
        mbar_wait_bounded(full_bar(i % STAGES), (i / STAGES) & 1, a.flags, WAIT_LIMIT_NS);
    // nor is a commit of the leader's that signals this CTA's barriers
    for (int i = max(0, g - STAGES); i < g; ++i)
      if (!mbar_wait(empty_bar(i % STAGES), (i / STAGES) & 1, a)) break;
  } else if (warp == 1 && leader) {
    // ---------------- MMA issuer (leader) ----------------
    const uint32_t base0 = smem_u32(smem);
    const uint64_t pd = operand_desc(base0), qd = operand_desc(base0 + C::P_BYTES), sd = scale_desc(base0 + C::P_BYTES + C::Q_BYTES);
    int s = 0, t = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs, ++t) {
      const int b = t % C::NACC;
      if (t >= C::NACC) ok = warp_wait(acce(b), ((t / C::NACC) & 1) ^ 1, a);
      if (!ok) break;
      const uint32_t acc = tmem + b * C::BN;
      asm volatile("tcgen05.fence::after_thread_sync;");
      int left = a.kbytes;
      for (int i = 0; i < n; ++i, left -= ROW_BYTES) {
        ok = warp_wait(full_bar(s), ph, a);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;");
        const uint32_t at = (uint32_t)(s * C::STAGE_BYTES) >> 4;  // the descriptors' address field counts 16 bytes
        const uint32_t sfp = tmem + C::BN + s * C::SF_COLS, sfq = sfp + C::SF_TILES * 4;
        const int steps = min(4, (left + 31) >> 5);
        if (elect_one()) {
          if (C::FP4) {
#pragma unroll
            for (int k = 0; k < C::SF_TILES; ++k) {
              copy_scales_pair(sfp + k * 4, sd + at + k * 32);
              copy_scales_pair(sfq + k * 8, sd + at + (C::PS_BYTES >> 4) + k * 32);
              copy_scales_pair(sfq + k * 8 + 4, sd + at + (2 * C::PS_BYTES >> 4) + k * 32);
            }
          }
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            if (kk >= steps) break;
            const int k = KIND == IC_NVFP4 ? kk : kk >> 1;
            const uint32_t id = KIND == IC_MXFP4 && (kk & 1) ? C::IDESC | (2u << 4) | (2u << 29) : C::IDESC;
            mma_pair<KIND>(acc, pd + at + kk * 2, qd + at + kk * 2, id, sfp + k * 4, sfq + k * 8, (i | kk) ? 1u : 0u);
          }
          mma_commit_pair(empty_bar(s));
          if (i == n - 1) mma_commit_pair(accf(b));
        }
        __syncwarp();
        if (++s == STAGES) {
          s = 0;
          ph ^= 1;
        }
      }
    }
    // products in flight end before their tensor memory is freed
    if (!ok && elect_one()) mma_commit_leader(last_bar);
    __syncwarp();
    mbar_wait_bounded(ok ? accf((t - 1) % C::NACC) : last_bar, ok ? ((t - 1) / C::NACC) & 1 : 0, a.flags, WAIT_LIMIT_NS);
  } else if (warp == 3) {
    // ---------------- factors of the coming tile (both CTAs) ----------------
    int t = 0;
    for (int tile = pair; tile < tiles; tile += pairs, ++t) {
      int p0, q0;
      place(tile, p0, q0);
      Factors& f = factors[t & 1];
      if (t >= 2 && !warp_wait(face(t & 1), ((t >> 1) & 1) ^ 1, a)) break;
      const int row0 = p0 + (int)rank * 128;
      float cf[8], cb[8], rf[4];
      load_strided(a.q_row, a.q_half ? IC_F16 : IC_F32, q0 + lane, a.qn, cf);
      load_strided(a.bias, a.bias_type, q0 + lane, a.qn, cb);
      load_strided(a.p_row, a.p_half ? IC_F16 : IC_F32, row0 + lane, a.pm, rf);
      int zp[8], sum[4];
      if (KIND == IC_INT8 && a.zp) {
#pragma unroll
        for (int i = 0; i < 8; ++i) zp[i] = q0 + i * 32 + lane < a.qn ? a.zp[q0 + i * 32 + lane] : 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = row0 + i * 32 + lane < a.pm ? a.sums[row0 + i * 32 + lane] : 0;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) zp[i] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] = 0;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f.col[i * 32 + lane] = cf[i];
        f.bias[i * 32 + lane] = cb[i];
        f.zp[i * 32 + lane] = zp[i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        f.row[i * 32 + lane] = rf[i];
        f.sum[i * 32 + lane] = sum[i];
      }
      mbar_arrive(facf(t & 1));
    }
  } else if (warp >= 4) {
    // ---------------- epilogue (both CTAs, own rows) ----------------
    const int q = warp & 3, h = (warp - 4) >> 2;
    unsigned char* out = out_smem + (warp - 4) * (32 * ROW_PITCH);
    int t = 0, tile = pair;
    for (; tile < tiles; tile += pairs, ++t) {
      int p0, q0;
      place(tile, p0, q0);
      const int row0 = p0 + (int)rank * 128 + q * 32, col0 = q0 + h * 128;
      const int b = t % C::NACC;
      if (!warp_wait(facf(t & 1), (t >> 1) & 1, a) || !warp_wait(accf(b), (t / C::NACC) & 1, a)) break;
      asm volatile("tcgen05.fence::after_thread_sync;");
      uint32_t acc[128];
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(b * C::BN + h * 128);
#pragma unroll
      for (int i = 0; i < 4; ++i) IC_TMEM_LD32(at + i * 32, acc + i * 32);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      asm volatile("tcgen05.fence::before_thread_sync;");
      __syncwarp();
      if (lane == 0) remote_arrive(map_to_rank(acce(b), 0));
      const Factors& f = factors[t & 1];
      if (a.out_type == IC_BF16) store_block<KIND, __nv_bfloat16>(a, acc, out, f, q * 32, h * 128, row0, col0, lane);
      else if (a.out_type == IC_F16) store_block<KIND, __half>(a, acc, out, f, q * 32, h * 128, row0, col0, lane);
      else store_block<KIND, float>(a, acc, out, f, q * 32, h * 128, row0, col0, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(face(t & 1));  // every lane has read the factors
    }
    for (; tile < tiles; tile += pairs) {  // a wait gave up: nor is a later tile of this warp's computed
      int p0, q0;
      place(tile, p0, q0);
      const int row0 = p0 + (int)rank * 128 + q * 32, col0 = q0 + h * 128;
      store_nan(a, (long long)row0 * a.ldy + col0, min(32, a.pm - row0), min(128, a.qn - col0), lane);
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;");
  __syncthreads();
  cluster_sync();  // no CTA leaves while its peer may still signal its barriers or read its operands
  if (warp == 2) {
    asm volatile("tcgen05.fence::after_thread_sync;");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS));
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(p);
    return EncodeTiledFn(nullptr);
  }();
  return fn;
}

int make_map(CUtensorMap* tm, const void* base, int64_t rows, int64_t kbytes, int64_t ld, int box_rows) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(IC_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[2] = {(cuuint64_t)kbytes, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)ld};
  cuuint32_t box[2] = {(cuuint32_t)ROW_BYTES, (cuuint32_t)box_rows};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(IC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) rows=%lld bytes=%lld ld=%lld", (int)r, (long long)rows,
                (long long)kbytes, (long long)ld);
  return IC_OK;
}

struct Operand {
  const void* codes;
  int64_t rows, ld;  // ld in bytes
  const uint8_t* scales;
  const void* row;
  int half;
};

template <int KIND, int BN>
int launch(const Operand& p, const Operand& q, LowpArgs a, int splits, cudaStream_t st) {
  using C = Cfg<KIND, BN>;
  static std::atomic<unsigned long long> done{0};
  IC_TRY(once_per_device(done, [] {
    IC_CUDA(cudaFuncSetAttribute(lowp_gemm_kernel<KIND, BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    return (int)IC_OK;
  }));
  CUtensorMap tp, tq;
  IC_TRY(make_map(&tp, p.codes, p.rows, a.kbytes, p.ld, BM));
  IC_TRY(make_map(&tq, q.codes, q.rows, a.kbytes, q.ld, BN));
  a.pm = (int)p.rows, a.qn = (int)q.rows;
  a.p_scales = p.scales, a.q_scales = q.scales;
  a.p_row = p.row, a.q_row = q.row, a.p_half = p.half, a.q_half = q.half;
  a.splits = splits;
  const int64_t tiles = cdiv(p.rows, BM) * cdiv(q.rows, BN);
  if (tiles * splits > INT32_MAX) return fail(IC_ERR_UNSUPPORTED, "matmul: too many tiles");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * splits), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)splits;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  IC_CUDA(cudaLaunchKernelEx(&cfg, lowp_gemm_kernel<KIND, BN>, tp, tq, a));
  IC_CHECK_LAUNCH();
  return IC_OK;
}

// block scales as [128-row tile][tile along K][512 bytes]; boxes of `tiles` x `atoms` tiles, zero beyond the matrix
int make_scale_map(CUtensorMap* tm, const uint8_t* base, int64_t row_tiles, int64_t ktiles, int tiles, int atoms) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return fail(IC_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  cuuint64_t dims[3] = {128, (cuuint64_t)ktiles, (cuuint64_t)row_tiles};
  cuuint64_t strides[2] = {512, (cuuint64_t)ktiles * 512};
  cuuint32_t box[3] = {128, (cuuint32_t)tiles, (cuuint32_t)atoms};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = fn(tm, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<uint8_t*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(IC_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d) for %lld scale tiles", (int)r, (long long)ktiles);
  return IC_OK;
}

template <int KIND>
int launch_pair(const Operand& p, const Operand& q, LowpArgs a, cudaStream_t st) {
  using C = PairCfg<KIND>;
  static std::atomic<unsigned long long> done{0};
  IC_TRY(once_per_device(done, [] {
    IC_CUDA(cudaFuncSetAttribute(lowp_pair_kernel<KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    return (int)IC_OK;
  }));
  CUtensorMap tp, tq, tps, tqs;
  IC_TRY(make_map(&tp, p.codes, p.rows, a.kbytes, p.ld, 128));
  IC_TRY(make_map(&tq, q.codes, q.rows, a.kbytes, q.ld, 128));
  if (C::FP4) {
    IC_TRY(make_scale_map(&tps, p.scales, cdiv(p.rows, 128), a.ktiles, C::SF_TILES, 1));
    IC_TRY(make_scale_map(&tqs, q.scales, cdiv(q.rows, 128), a.ktiles, C::SF_TILES, 2));
  } else {
    tps = tp, tqs = tq;
  }
  a.pm = (int)p.rows, a.qn = (int)q.rows;
  a.p_row = p.row, a.q_row = q.row, a.p_half = p.half, a.q_half = q.half;
  const int64_t tiles = cdiv(p.rows, 256) * cdiv(q.rows, C::BN);
  if (tiles > INT32_MAX / 2) return fail(IC_ERR_UNSUPPORTED, "matmul: too many tiles");
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(384, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  // as many pairs as the device holds at once (an odd SM of a GPC has no partner)
  static std::atomic<int> resident[64];
  int dev = 0;
  IC_CUDA(cudaGetDevice(&dev));
  int pairs = resident[dev & 63].load();
  if (!pairs) {
    cfg.gridDim = dim3(2, 1, 1);
    IC_CUDA(cudaOccupancyMaxActiveClusters(&pairs, lowp_pair_kernel<KIND>, &cfg));
    if (pairs < 1) return fail(IC_ERR_CUDA, "matmul: no CTA pair fits the device");
    resident[dev & 63].store(pairs);
  }
  cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, pairs)), 1, 1);
  IC_CUDA(cudaLaunchKernelEx(&cfg, lowp_pair_kernel<KIND>, tp, tq, tps, tqs, a));
  IC_CHECK_LAUNCH();
  return IC_OK;
}

// How a product is cut: tile width, orientation and K split
struct Plan {
  int bn;      // 256-row pairs when 0
  bool swap;   // the weights take the 128-row side
  int splits;
  double clocks;
};

// Estimated SM clocks of a one-CTA plan.  A stage takes the longer of its
// products (BN/2 clocks for each of four) and its loads (63 bytes a clock and
// SM, measured with all SMs loading from L2); a CTA's start, first loads and
// epilogue take about 4000 clocks and per column 8 (aligned rows of y), 45 (other
// rows) or 20 (weights in P), a split's exchange 2500 and 16 a column.
// (Over 24 products from 1 x 4096 x 4096 to 4607 x 16383 x 4096, every plan
// timed: 21 choices are within 7% of the fastest, the worst 21% off.)
template <int KIND, int BN>
void consider(Plan& best, int64_t pm, int64_t qn, int64_t stages, bool swap, bool aligned) {
  using C = Cfg<KIND, BN>;
  const int64_t tiles = cdiv(pm, BM) * cdiv(qn, BN);
  for (int s = 1; s <= MAX_SPLIT && s <= stages; s *= 2) {
    const int64_t ctas = tiles * s, waves = cdiv(ctas, 148 * C::CTAS);
    const int per_sm = (int)std::min<int64_t>(C::CTAS, cdiv(ctas, 148));
    const double stage = std::max(2.0 * BN, C::STAGE_BYTES / 63.0) * per_sm;
    const double store = swap ? 20 : aligned ? 8 : 45, ends = 4000 + store * BN / s + (s > 1 ? 2500 + 16.0 * BN : 0);
    const double clocks = waves * ((double)cdiv(stages, s) * stage + ends * (per_sm > 1 ? 1.5 : 1));  // two CTAs share an SM's ends too
    if (clocks < best.clocks) best = Plan{BN, swap, s, clocks};
  }
}

template <int KIND>
Plan plan(int64_t m, int64_t n, int64_t stages, bool aligned) {
  // pairs: 620 clocks a stage and 3000 between tiles (nvfp4's, for all kinds: int8 takes 530), or an epilogue of
  // element stores; a longer start (measured)
  Plan best{0, false, 1, cdiv(cdiv(m, 256) * cdiv(n, 256), 74) * std::max(stages * 620.0 + 3000, aligned ? 0.0 : 18000.0) + 5000};
  for (int swap = 0; swap < 2; ++swap) {
    const int64_t pm = swap ? n : m, qn = swap ? m : n;
    if (qn <= 16) consider<KIND, 16>(best, pm, qn, stages, swap, aligned);
    if (qn <= 32) consider<KIND, 32>(best, pm, qn, stages, swap, aligned);
    consider<KIND, 64>(best, pm, qn, stages, swap, aligned);
    consider<KIND, 128>(best, pm, qn, stages, swap, aligned);
    consider<KIND, 192>(best, pm, qn, stages, swap, aligned);
    consider<KIND, 256>(best, pm, qn, stages, swap, aligned);
  }
  return best;
}

// The plan of this thread's next product, where the self-test gives one (splits > 0)
thread_local Plan g_plan{0, false, 0, 0.0};

// a plan that the kernels can run: narrow tiles cover all rows of Q, every split has a stage, pairs know neither
bool possible(const Plan& b, int64_t qn, int64_t stages) {
  return b.bn ? b.splits <= stages && (b.bn > 32 || qn <= b.bn) : b.splits == 1 && !b.swap;
}

// x [m, k] times w [n, k]^T
template <int KIND>
int matmul(const Operand& x, const Operand& w, LowpArgs a, cudaStream_t st) {
  const int64_t size = a.out_type == IC_F32 ? 4 : 2;
  const bool aligned = ((reinterpret_cast<uintptr_t>(a.y) | (uintptr_t)(a.ldy * size)) & 15) == 0;
  const int64_t stages = cdiv(a.kbytes, ROW_BYTES);
  Plan b = g_plan;
  g_plan.splits = 0;
  if (!b.splits) b = plan<KIND>(x.rows, w.rows, stages, aligned);
  else if (!possible(b, b.swap ? x.rows : w.rows, stages)) return fail(IC_ERR_INVALID, "selftest: no such plan of this product");
  a.swap = b.swap;
  const Operand &p = b.swap ? w : x, &q = b.swap ? x : w;
  switch (b.bn) {
    case 16: return launch<KIND, 16>(p, q, a, b.splits, st);
    case 32: return launch<KIND, 32>(p, q, a, b.splits, st);
    case 64: return launch<KIND, 64>(p, q, a, b.splits, st);
    case 128: return launch<KIND, 128>(p, q, a, b.splits, st);
    case 192: return launch<KIND, 192>(p, q, a, b.splits, st);
    case 256: return launch<KIND, 256>(p, q, a, b.splits, st);
    default: return launch_pair<KIND>(x, w, a, st);
  }
}

int check_product(const char* what, int64_t m, int64_t n, int64_t k, const void* bias, int bias_dtype, int out_dtype,
                  const void* y, int64_t ldy) {
  if (m < 0 || n < 0 || k <= 0 || ldy < n) return fail(IC_ERR_INVALID, "%s: bad shape", what);
  if (m > INT32_MAX / 2 || n > INT32_MAX / 2 || k > INT32_MAX / 2) return fail(IC_ERR_UNSUPPORTED, "%s: size", what);
  if (out_dtype < IC_F32 || out_dtype > IC_BF16 || (bias && (bias_dtype < IC_F32 || bias_dtype > IC_BF16)))
    return fail(IC_ERR_INVALID, "%s: unknown dtype", what);
  if (m > 0 && n > 0 && !y) return fail(IC_ERR_INVALID, "%s: null pointer", what);
  return IC_OK;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// The device status word.  Where none exists yet it is this file's own static
// one: allocating it would end a stream capture that the first product is part of.
__device__ unsigned g_lowp_flags;
unsigned* status_word() {
  static std::atomic<unsigned long long> done{0};
  const int r = once_per_device(done, [] {
    int dev = 0;
    void* p = nullptr;
    IC_CUDA(cudaGetDevice(&dev));
    IC_CUDA(cudaGetSymbolAddress(&p, g_lowp_flags));
    register_device_flags(dev, static_cast<unsigned*>(p));
    return (int)IC_OK;
  });
  return r == IC_OK ? device_flags() : nullptr;
}

// What the next product of this thread is to load, and how long its waits last
struct Stall {
  int loads = INT32_MAX;
  unsigned wait_ns = WAIT_LIMIT_NS;
};
thread_local Stall g_stall;

int set_waits(LowpArgs& a) {
  a.flags = status_word();
  if (!a.flags) return fail(IC_ERR_CUDA, "device status word unavailable");
  a.loads = g_stall.loads, a.wait_ns = g_stall.wait_ns;
  g_stall = Stall{};
  return IC_OK;
}

}  // namespace
}  // namespace ic

extern "C" int ic_selftest_matmul_stall(int stages, unsigned long long limit_ns) {
  using namespace ic;
  if (stages < 0 || limit_ns < 100000ull || limit_ns > WAIT_LIMIT_NS)
    return fail(IC_ERR_INVALID, "selftest: stages must not be negative, the wait limit in [0.1 ms, 2 s]");
  g_stall = Stall{stages, (unsigned)limit_ns};
  return IC_OK;
}

extern "C" int ic_selftest_matmul_plan(int width, int swap, int splits) {
  using namespace ic;
  bool ok = width == 0 || width == 192 || (width >= 16 && width <= 256 && !(width & (width - 1)));
  ok = ok && swap >= 0 && swap <= 1 && splits >= 1 && splits <= MAX_SPLIT && !(splits & (splits - 1));
  if (!ok) return fail(IC_ERR_INVALID, "selftest: no such plan");
  g_plan = Plan{width, swap != 0, splits, 0.0};
  return IC_OK;
}

extern "C" int ic_fp4_matmul(const uint8_t* a_packed, const uint8_t* a_scales, const float* a_row_scale,
                             const uint8_t* b_packed, const uint8_t* b_scales, const float* b_row_scale, int fmt,
                             int64_t m, int64_t n, int64_t kp, const void* bias, int bias_dtype, int out_dtype, void* y,
                             int64_t ldy, void* stream) {
  using namespace ic;
  if (fmt != IC_MXFP4 && fmt != IC_NVFP4) return fail(IC_ERR_INVALID, "fp4_matmul: unknown format %d", fmt);
  IC_TRY(check_product("fp4_matmul", m, n, kp, bias, bias_dtype, out_dtype, y, ldy));
  if (kp % 32) return fail(IC_ERR_INVALID, "fp4_matmul: kp must be a multiple of 32");
  if (m == 0 || n == 0) return IC_OK;
  if (!a_packed || !a_scales || !b_packed || !b_scales || (fmt == IC_NVFP4 && (!a_row_scale || !b_row_scale)))
    return fail(IC_ERR_INVALID, "fp4_matmul: null pointer");
  if (!aligned16(a_packed) || !aligned16(a_scales) || !aligned16(b_packed) || !aligned16(b_scales))
    return fail(IC_ERR_INVALID, "fp4_matmul: codes and scales must be 16-byte aligned");
  LowpArgs a{};
  a.kbytes = (int)(kp / 2);
  a.ktiles = (int)fp4_ktiles(fmt, kp);
  a.bias = bias, a.bias_type = bias_dtype, a.y = y, a.ldy = ldy, a.out_type = out_dtype;
  IC_TRY(set_waits(a));
  const bool nv = fmt == IC_NVFP4;
  const Operand x{a_packed, m, kp / 2, a_scales, nv ? a_row_scale : nullptr, 0};
  const Operand w{b_packed, n, kp / 2, b_scales, nv ? b_row_scale : nullptr, 0};
  return nv ? matmul<IC_NVFP4>(x, w, a, (cudaStream_t)stream) : matmul<IC_MXFP4>(x, w, a, (cudaStream_t)stream);
}

extern "C" int ic_int8_matmul(const int8_t* codes, int64_t lda, const float* scales, const int32_t* sums,
                              const int8_t* w_codes, int64_t ldw, const uint16_t* w_scales_f16, const int8_t* w_zp,
                              int64_t m, int64_t n, int64_t k, const void* bias, int bias_dtype, int out_dtype, void* y,
                              int64_t ldy, void* stream) {
  using namespace ic;
  IC_TRY(check_product("int8_matmul", m, n, k, bias, bias_dtype, out_dtype, y, ldy));
  // |sum a*w| <= 2^14 k, and with zero-points |sum a*(w - zp)| and zp * sum a on top of it
  if (k > (w_zp ? 65535 : 131071)) return fail(IC_ERR_UNSUPPORTED, "int8_matmul: int32 sums hold k up to %d", w_zp ? 65535 : 131071);
  if (m == 0 || n == 0) return IC_OK;
  if (!codes || !scales || !w_codes || !w_scales_f16 || (w_zp && !sums)) return fail(IC_ERR_INVALID, "int8_matmul: null pointer");
  if (lda < k || ldw < k || lda % 16 || ldw % 16 || !aligned16(codes) || !aligned16(w_codes))
    return fail(IC_ERR_INVALID, "int8_matmul: rows of codes must be 16-byte aligned, with pitches of a multiple of 16");
  LowpArgs a{};
  a.kbytes = (int)k;
  a.zp = w_zp, a.sums = sums;
  a.bias = bias, a.bias_type = bias_dtype, a.y = y, a.ldy = ldy, a.out_type = out_dtype;
  IC_TRY(set_waits(a));
  const Operand x{codes, m, lda, nullptr, scales, 0};
  const Operand w{w_codes, n, ldw, nullptr, w_scales_f16, 1};
  return matmul<IC_INT8>(x, w, a, (cudaStream_t)stream);
}
