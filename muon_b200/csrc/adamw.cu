// Multi-tensor AdamW: see adamw.h. All kernels here are bound by HBM traffic.
#include "adamw.h"

#include "common.cuh"
#include "elementwise.h"
#include "ns_gemm.h"
#include "profiling.h"

#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>
#include <initializer_list>
#include <type_traits>

namespace mb {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// ---------------------------------------------------------------------------
// N consecutive elements of T as floats: 16 or 32 bytes, on a boundary of as many.
// 32 bytes go in one access: two of 16 would each touch every sector of the row and move half of it.
// What a step reads and writes once (ONCE) is the first to leave L2, so that the gradients a norm has
// read before it stay there longer.
// ---------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b);
template <>
__device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
template <>
__device__ __forceinline__ void unpack2<__half>(uint32_t w, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) { return pack_bf16x2(a, b); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int N>
struct Raw {  // the words of N elements, as loaded
  static constexpr int kWords = N * (int)sizeof(T) / 16;
  static_assert(kWords == 1 || kWords % 2 == 0, "16 bytes or pieces of 32");
  uint4 w[kWords];
  template <bool ONCE = false>
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords == 1) {
      w[0] = __ldcs(reinterpret_cast<const uint4*>(p));
    } else {
#pragma unroll
      for (int k = 0; k + 1 < kWords; k += 2) {
        const uint4* q = reinterpret_cast<const uint4*>(p) + k;
#define MB_LOAD32(OP)                                                                                              \
  asm volatile(OP " {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"                                                       \
               : "=r"(w[k].x), "=r"(w[k].y), "=r"(w[k].z), "=r"(w[k].w), "=r"(w[k + 1].x), "=r"(w[k + 1].y),       \
                 "=r"(w[k + 1].z), "=r"(w[k + 1].w)                                                                \
               : "l"(q)                                                                                            \
               : "memory")
        if constexpr (ONCE) MB_LOAD32("ld.global.L2::evict_first.v8.b32");
        else MB_LOAD32("ld.global.v8.b32");
#undef MB_LOAD32
      }
    }
  }
  template <bool ONCE = false>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kWords == 1) {
      __stcs(reinterpret_cast<uint4*>(p), w[0]);
    } else {
#pragma unroll
      for (int k = 0; k + 1 < kWords; k += 2) {
        uint4* q = reinterpret_cast<uint4*>(p) + k;
#define MB_STORE32(OP)                                                                                             \
  asm volatile(OP " [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(q), "r"(w[k].x), "r"(w[k].y), "r"(w[k].z),      \
               "r"(w[k].w), "r"(w[k + 1].x), "r"(w[k + 1].y), "r"(w[k + 1].z), "r"(w[k + 1].w)                     \
               : "memory")
        if constexpr (ONCE) MB_STORE32("st.global.L2::evict_first.v8.b32");
        else MB_STORE32("st.global.v8.b32");
#undef MB_STORE32
      }
    }
  }
  __device__ __forceinline__ void unpack(float (&v)[N]) const {
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const uint32_t u[4] = {w[k].x, w[k].y, w[k].z, w[k].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) v[4 * k + j] = __uint_as_float(u[j]);
        else unpack2<T>(u[j], v[8 * k + 2 * j], v[8 * k + 2 * j + 1]);
      }
    }
  }
  __device__ __forceinline__ void pack(const float (&v)[N]) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      uint32_t u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) u[j] = __float_as_uint(v[4 * k + j]);
        else u[j] = pack2<T>(v[8 * k + 2 * j], v[8 * k + 2 * j + 1]);
      }
      w[k] = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
  __device__ __forceinline__ void unpack(float2 (&v)[N / 2]) const {
    float x[N];
    unpack(x);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) v[j] = make_float2(x[2 * j], x[2 * j + 1]);
  }
  __device__ __forceinline__ void pack(const float2 (&v)[N / 2]) {
    float x[N];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
      x[2 * j] = v[j].x;
      x[2 * j + 1] = v[j].y;
    }
    pack(x);
  }
};

// Two float32 operations in one instruction, one rounding each.
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
// a + b where a is a product: as a multiply-add by a 1 that the compiler does not know (the assembler
// fuses a paired product and a paired sum into one operation with one rounding, unlike single ones).
__device__ __forceinline__ float2 add2(float2 a, float2 b, float one) { return __ffma2_rn(a, both(one), b); }

__device__ __forceinline__ float sqrt_approx(float x) {  // relative error at most 2^-23
  float r;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// Index of the table entry whose range of chunks holds `chunk` (start[0] = 0, ascending).
template <typename S>
__device__ __forceinline__ int find_tensor(const S& start, int count, int chunk) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (chunk >= start[mid]) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Tensors that start anywhere are handled in aligned pieces from their `head` on, where the lists of a
// tensor are all aligned at one element (as in tensors packed one behind the other).
constexpr unsigned char kNoHead = 255;

// A step often follows a norm of the same gradients: each launch starts with the last of its tensors, whose
// gradients are still in L2 (a call with more tensors than a table holds launches its tables in the order of the
// lists). Norm and step of 218M bf16 weights with 8-bit moments take 412 us so, 419 in the order of the lists and with
// ordinary accesses; 100M bf16 weights with float32 moments 355 and 362, 128 float32 filters (47M) 225 and 229.
__device__ __forceinline__ int from_the_end() { return (int)(gridDim.x - 1 - blockIdx.x); }

struct AdamWConsts {
  float b1, w1, b2, w2;  // float(beta), float(1 - beta)
  float eps, decay;      // decay = float(1 - lr * weight_decay)
  float one;             // 1 (see add2)
  const float* grad_scale;
  int count;
};

// p (1 - lr wd) - (lr / c1) m / (sqrt(v) / sqrt(c2) + eps). The square root and the quotient are the
// hardware's approximations (about 2^-22 together): they only scale an update that is itself a
// small fraction of p.
__device__ __forceinline__ float moved(float p, float m, float v, float decay, float step, float rs, float eps) {
  const float den = fmaf(sqrt_approx(v), rs, eps);
  return fmaf(-step, __fdividef(m, den), p * decay);
}

// The factor that every gradient is multiplied by. A factor that is not finite (the norm was not)
// means: leave everything as it is. Waits for the kernel before this one, which may have left the factor
// (launch_after); nothing is read or written before.
__device__ __forceinline__ bool read_factor(const float* grad_scale, float& f) {
  griddep_wait();
  f = grad_scale ? *grad_scale : 1.f;
  return fabsf(f) <= 3.402823466e38f;
}

// ---------------------------------------------------------------------------
// AdamW with 32-bit moments.
//   g' = g f;  m = b1 m + (1-b1) g';  v = b2 v + (1-b2) g'^2
//   p  = p (1 - lr wd) - (lr/c1) m / (sqrt(v)/sqrt(c2) + eps)
// in float32 registers, p rounded once when it is stored. With a master weight p is the master and
// the parameter receives its rounded copy. Bound by HBM: 872M bf16 weights 2791 us, 6.9 TB/s. Lists that are never
// aligned together (packed parameters with moments of their own, say) go element by element: 100M weights 496 us
// with bf16 and 472 with float32 parameters (4.4 and 5.9 TB/s), where aligned ones take 322 and 407.
// ---------------------------------------------------------------------------
template <int CAP>
struct AdamW32Args {
  AdamWConsts c;
  void* p[CAP];
  float* w[CAP];
  const void* g[CAP];
  float* m[CAP];
  float* v[CAP];
  long long numel[CAP];
  float step[CAP], rs[CAP];
  int start[CAP + 1];
  unsigned char head[CAP];  // elements before the first that is aligned in every list; kNoHead: none is
};

template <typename P>
constexpr int kVec32 = sizeof(P) == 4 ? 4 : 8;
// One vector a thread and no loop: four streams in and three out keep enough bytes in flight by themselves,
// and short-lived blocks leave no tail. Four layers of bf16 weights, 872M: 2791 us, 2826, 2859, 2914 with 1, 2, 4, 8
// vectors a thread; 128 float32 filters, 47M: 193, 196, 200, 203.
template <typename P>
constexpr int kChunk32 = kThreads * kVec32<P>;

template <typename P, typename G, bool MASTER, int CAP>
__global__ void __launch_bounds__(kThreads)
adamw32_kernel(const __grid_constant__ AdamW32Args<CAP> a) {
  constexpr int V = kVec32<P>;
  float f;
  if (!read_factor(a.c.grad_scale, f)) return;
  const int block = from_the_end();
  const int t = find_tensor(a.start, a.c.count, block);
  const int head = a.head[t] == kNoHead ? 0 : a.head[t];
  const int chunk = block - a.start[t];
  const long long base = (long long)chunk * kChunk32<P> + head;
  const long long left = a.numel[t] - base;
  P* p = static_cast<P*>(a.p[t]) + base;
  float* w = MASTER ? a.w[t] + base : nullptr;
  const G* g = static_cast<const G*>(a.g[t]) + base;
  float* m = a.m[t] + base;
  float* v = a.v[t] + base;
  const float step = a.step[t], rs = a.rs[t];
  const AdamWConsts c = a.c;
  const auto one = [&](float& pj, float gj, float& mj, float& vj) {
    gj *= f;
    mj = fmaf(gj, c.w1, mj * c.b1);
    vj = fmaf(gj * gj, c.w2, vj * c.b2);
    pj = moved(pj, mj, vj, c.decay, step, rs, c.eps);
  };
  int done = 0;  // elements of the chunk that the vector loop covers
  if (a.head[t] != kNoHead) {
    done = left >= kChunk32<P> ? kChunk32<P> : (int)left / V * V;
    const int i = threadIdx.x * V;
    if (i < done) {
      Raw<P, V> rp;
      Raw<float, V> rw, rm, rv;
      Raw<G, V> rg;
      if constexpr (MASTER) rw.template load<true>(w + i);
      else rp.template load<true>(p + i);
      rg.template load<true>(g + i);
      rm.template load<true>(m + i);
      rv.template load<true>(v + i);
      float pj[V], gj[V], mj[V], vj[V];
      if constexpr (MASTER) rw.unpack(pj);
      else rp.unpack(pj);
      rg.unpack(gj);
      rm.unpack(mj);
      rv.unpack(vj);
#pragma unroll
      for (int j = 0; j < V; ++j) one(pj[j], gj[j], mj[j], vj[j]);
      rm.pack(mj);
      rm.template store<true>(m + i);
      rv.pack(vj);
      rv.template store<true>(v + i);
      if constexpr (MASTER) {
        rw.pack(pj);
        rw.template store<true>(w + i);
      }
      rp.pack(pj);
      rp.template store<true>(p + i);
    }
  }
  const auto single = [&](int i) {
    float pj = MASTER ? w[i] : to_float<P>(p[i]), mj = m[i], vj = v[i];
    one(pj, to_float<G>(g[i]), mj, vj);
    m[i] = mj;
    v[i] = vj;
    if (MASTER) w[i] = pj;
    p[i] = from_float<P>(pj);
  };
  const int end = left < kChunk32<P> ? (int)left : kChunk32<P>;
  for (int i = done + threadIdx.x; i < end; i += kThreads) single(i);
  if (chunk == 0 && (int)threadIdx.x < head) single((int)threadIdx.x - head);
}

// ---------------------------------------------------------------------------
// 8-bit moments. A block of kStateBlock consecutive elements shares a float32 scale per moment; one
// warp handles a block, eight elements a lane.
//   first moment   e4m3, value = code * scale, scale = amax / 448, nearest even
//   second moment  5 exponent and 3 mantissa bits without a sign: value = scale * w(c), where w(c) is the
//                  float whose bits are (c + 768) << 20, i.e. 2^((c >> 3) - 31) (1 + (c & 7) / 8);
//                  scale = amax / 1.875 = amax / w(255)
// Neither needs a table. Unsigned: a second moment has no sign, so its mantissa gets that bit; 32
// binades hold gradients that differ by 2^16 within a block; code 0 stands for 2^-31, so no element of a
// block that is in use ever divides by nothing.
//
// What is rounded to a code, and the code, are a function of float32 operations with one rounding each
// (no fused multiply-add): the same step written in any float32 arithmetic gives the same codes.
//
// The second moment is rounded stochastically in a step: with beta2 = 0.999 a step moves it by a
// thousandth, a code is 6 to 12 percent wide, and rounding to nearest would never move it.
// x = v * (1.875 / amax) as bits, plus 20 random bits, cut at bit 20: right on average, exactly.
// ---------------------------------------------------------------------------
constexpr float kE4m3Max = 448.f, kSqMax = 1.875f;
constexpr float kTinyAvg = 0x1p-110f, kTinySq = 0x1p-120f;  // below: the block counts as zero

template <int KIND>
__device__ __forceinline__ float block_scale(float amax) {
  constexpr float top = KIND == STATE_EXP_AVG ? kE4m3Max : kSqMax;
  return amax < (KIND == STATE_EXP_AVG ? kTinyAvg : kTinySq) ? 0.f : __fmul_rn(amax, 1.f / top);
}
template <int KIND>
__device__ __forceinline__ float block_factor(float amax) {
  constexpr float top = KIND == STATE_EXP_AVG ? kE4m3Max : kSqMax;
  return amax < (KIND == STATE_EXP_AVG ? kTinyAvg : kTinySq) ? 0.f : __fdiv_rn(top, amax);
}

// Largest |x| over the warp of the largest of each lane, by the bits: a NaN is above everything.
__device__ __forceinline__ float warp_max(uint32_t bits) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, bits));
}
__device__ __forceinline__ uint32_t amax_bits(const float2 (&x)[4]) {
  float m;
  asm("{\n\tmax.NaN.abs.f32 %0, %1, %2, %3;\n\tmax.NaN.abs.f32 %0, %0, %4, %5;\n\tmax.NaN.abs.f32 %0, %0, %6, %7;\n\t"
      "max.NaN.abs.f32 %0, %0, %8, %8;\n\t}"
      : "=&f"(m)
      : "f"(x[0].x), "f"(x[0].y), "f"(x[1].x), "f"(x[1].y), "f"(x[2].x), "f"(x[2].y), "f"(x[3].x), "f"(x[3].y));
  return __float_as_uint(m);
}
// The same for values that have no sign bit (a sum of squares; an arithmetic NaN has none either).
__device__ __forceinline__ uint32_t amax_bits_unsigned(const float2 (&x)[4]) {
  const uint32_t a = __vimax3_u32(__float_as_uint(x[0].x), __float_as_uint(x[0].y), __float_as_uint(x[1].x));
  const uint32_t b = __vimax3_u32(__float_as_uint(x[1].y), __float_as_uint(x[2].x), __float_as_uint(x[2].y));
  return __vimax3_u32(a, b, max(__float_as_uint(x[3].x), __float_as_uint(x[3].y)));
}

__device__ __forceinline__ uint32_t e4m3_pair(float2 x) { return __nv_cvt_float2_to_fp8x2(x, __NV_SATFINITE, __NV_E4M3); }
__device__ __forceinline__ float2 e4m3_values(uint32_t pair) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// (code + 768) << 20 of byte j of a word: the offset's bits lie above the code's.
template <int J>
__device__ __forceinline__ float sq_value(uint32_t word) {
  const uint32_t c = J < 3 ? word << (J < 3 ? 20 - 8 * J : 0) : word >> 4;
  return __uint_as_float((c & 0x0ff00000u) | 0x30000000u);
}
// SIGNED: x may be -0 or negative, which is cut to the smallest code (with the sign bit among the others a
// negative x close to zero would come out as the largest). A step's sums of squares have no sign.
template <bool SIGNED>
__device__ __forceinline__ int sq_cut(float x, uint32_t r) {
  const uint32_t bits = SIGNED ? (uint32_t)max((int)__float_as_uint(x), 0) : __float_as_uint(x);
  return (int)(bits + r - 0x30000000u) >> 20;
}
// Two integers clamped to 0..255 as bytes 0 and 1, bytes 2 and 3 from the low half of `high`.
__device__ __forceinline__ uint32_t pack_bytes(int b1, int b0, uint32_t high) {
  uint32_t d;
  asm("cvt.pack.sat.u8.s32.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(b1), "r"(b0), "r"(high));
  return d;
}

// Eight codes of a moment <-> floats.
template <int KIND>
__device__ __forceinline__ void decode8(uint2 w, float2 (&x)[4]) {  // in units of the scale
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t u = h ? w.y : w.x;
    if constexpr (KIND == STATE_EXP_AVG) {
      x[2 * h] = e4m3_values(u & 0xffffu);
      x[2 * h + 1] = e4m3_values(u >> 16);
    } else {
      x[2 * h] = make_float2(sq_value<0>(u), sq_value<1>(u));
      x[2 * h + 1] = make_float2(sq_value<2>(u), sq_value<3>(u));
    }
  }
}
template <int KIND>
__device__ __forceinline__ void decode8(uint2 w, float scale, float2 (&x)[4]) {
  decode8<KIND>(w, x);
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = mul2(x[j], both(scale));
}
template <int KIND, bool SIGNED = false>
__device__ __forceinline__ uint2 encode8(const float2 (&x)[4], float inv, const uint32_t (&r)[8]) {
  const float2 f = make_float2(inv, inv);
  float2 y[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) y[j] = mul2(x[j], f);
  if constexpr (KIND == STATE_EXP_AVG) {
    return make_uint2(e4m3_pair(y[0]) | e4m3_pair(y[1]) << 16, e4m3_pair(y[2]) | e4m3_pair(y[3]) << 16);
  } else {
    uint32_t u[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      u[h] = pack_bytes(sq_cut<SIGNED>(y[2 * h].y, r[4 * h + 1]), sq_cut<SIGNED>(y[2 * h].x, r[4 * h]),
                        pack_bytes(sq_cut<SIGNED>(y[2 * h + 1].y, r[4 * h + 3]), sq_cut<SIGNED>(y[2 * h + 1].x, r[4 * h + 2]), 0u));
    return make_uint2(u[0], u[1]);
  }
}
// One code.
template <int KIND>
__device__ __forceinline__ float decode1(uint32_t c, float scale) {
  return __fmul_rn(KIND == STATE_EXP_AVG ? e4m3_values(c).x : sq_value<0>(c), scale);
}
__device__ __forceinline__ uint8_t byte_of(uint2 w, int j) { return (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3))); }

// Factors that bring the largest magnitudes of a block to the largest codes: the two halves of the warp
// compute one each (a division is the longest single thing a block needs).
__device__ __forceinline__ void both_factors(float m_amax, float v_amax, int lane, float& m_inv, float& v_inv) {
  const bool sq = lane >= 16;
  const float amax = sq ? v_amax : m_amax;
  const float inv = amax < (sq ? kTinySq : kTinyAvg) ? 0.f : __fdiv_rn(sq ? kSqMax : kE4m3Max, amax);
  m_inv = __shfl_sync(0xffffffffu, inv, 0);
  v_inv = __shfl_sync(0xffffffffu, inv, 16);
}

// 32 random bits for the four elements 4 * word .. 4 * word + 3; element j takes the low 20 bits of
// the word turned right by 8 j. The multipliers are the prime 0x9E3779B1, which lies near the fractional part of
// the golden ratio, and the fractional parts of the square roots of 2 and 3, in 32 bits; in the key those of the
// square roots of 5 (made odd) and 3.
__device__ __forceinline__ uint32_t random_word(uint32_t word, uint32_t key) {
  uint32_t h = word * 0x9E3779B1u + key;
  h = (h ^ (h >> 16)) * 0x6A09E667u;
  h = (h ^ (h >> 15)) * 0xBB67AE85u;
  return h ^ (h >> 16);
}
__device__ __forceinline__ uint32_t random_bits(uint32_t h, int j) { return __funnelshift_r(h, h, 8 * j) & 0xfffffu; }
inline uint32_t random_key(uint32_t seed, int64_t step) { return seed * 0x3C6EF373u + (uint32_t)step * 0xBB67AE85u; }

template <int CAP>
struct AdamW8Args {
  AdamWConsts c;
  void* p[CAP];
  float* w[CAP];
  const void* g[CAP];
  uint8_t* m[CAP];
  float* ms[CAP];
  uint8_t* v[CAP];
  float* vs[CAP];
  long long numel[CAP];
  float step[CAP], rs[CAP];
  uint32_t key[CAP];
  int start[CAP + 1];
  unsigned char vec_ok[CAP];
  int per_warp;  // blocks of a warp's task, 1 to 32
};

constexpr int kBlocksPerSm8 = 3;

// What a warp needs of a tensor.
template <typename P, typename G>
struct Tensor8 {
  P* p;
  float* w;
  const G* g;
  uint8_t *m, *v;
  float *ms, *vs;
  long long numel;
  float step, rs;
  uint32_t key;
};

// New moments and parameters of a lane's eight elements. The moments as the format prescribes, one
// rounding per operation, two elements per instruction; the update with the hardware's reciprocal
// (eps is at least 1e-16, so the denominator is a normal number and a second moment too small for
// one does not matter).
template <typename T>
__device__ __forceinline__ void step8(const AdamWConsts& c, const T& t, float f, float2 (&p)[4], float2 (&g)[4],
                                      float2 (&m)[4], float2 (&v)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    g[j] = mul2(g[j], both(f));
    m[j] = add2(mul2(m[j], both(c.b1)), mul2(g[j], both(c.w1)), c.one);
    v[j] = add2(mul2(v[j], both(c.b2)), mul2(mul2(g[j], g[j]), both(c.w2)), c.one);
    float2 root, inverse;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root.x) : "f"(v[j].x));
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(root.y) : "f"(v[j].y));
    const float2 den = __ffma2_rn(root, both(t.rs), both(c.eps));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse.x) : "f"(den.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse.y) : "f"(den.y));
    p[j] = __ffma2_rn(both(-t.step), mul2(m[j], inverse), mul2(p[j], both(c.decay)));
  }
}

// A block that is cut short by the tensor's end, or that does not start on a 16-byte boundary: a lane
// takes every 32nd element.
template <typename P, typename G, bool MASTER>
__device__ __forceinline__ void ragged_block8(const AdamWConsts& c, const Tensor8<P, G>& t, float f, long long b) {
  const int lane = threadIdx.x & 31;
  const long long base = b * kStateBlock + lane;
  const int n = (int)min((long long)kStateBlock, t.numel - b * kStateBlock) - lane;  // this lane's: j with 32 j < n
  const float ms = t.ms[b], vs = t.vs[b];
  float2 pj[4], gj[4], mj[4], vj[4];
  uint32_t r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool in = 32 * j < n;
    const long long i = base + 32 * j;
    float& pe = j & 1 ? pj[j / 2].y : pj[j / 2].x;
    float& ge = j & 1 ? gj[j / 2].y : gj[j / 2].x;
    float& me = j & 1 ? mj[j / 2].y : mj[j / 2].x;
    float& ve = j & 1 ? vj[j / 2].y : vj[j / 2].x;
    pe = in ? (MASTER ? t.w[i] : to_float<P>(t.p[i])) : 0.f;
    ge = in ? to_float<G>(t.g[i]) : 0.f;
    me = in ? decode1<STATE_EXP_AVG>(t.m[i], ms) : 0.f;
    ve = in ? decode1<STATE_EXP_AVG_SQ>(t.v[i], vs) : 0.f;
    r[j] = random_bits(random_word((uint32_t)(i >> 2), t.key), (int)(i & 3));
  }
  step8(c, t, f, pj, gj, mj, vj);
  const float m_amax = warp_max(amax_bits(mj)), v_amax = warp_max(amax_bits_unsigned(vj));
  float m_inv, v_inv;
  both_factors(m_amax, v_amax, lane, m_inv, v_inv);
  if (lane == 0) {
    t.ms[b] = block_scale<STATE_EXP_AVG>(m_amax);
    t.vs[b] = block_scale<STATE_EXP_AVG_SQ>(v_amax);
  }
  const uint2 cm = encode8<STATE_EXP_AVG>(mj, m_inv, r);
  const uint2 cv = encode8<STATE_EXP_AVG_SQ>(vj, v_inv, r);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const long long i = base + 32 * j;
    if (32 * j < n) {
      const float pe = j & 1 ? pj[j / 2].y : pj[j / 2].x;
      t.m[i] = byte_of(cm, j);
      t.v[i] = byte_of(cv, j);
      if (MASTER) t.w[i] = pe;
      t.p[i] = from_float<P>(pe);
    }
  }
}

// (Through L1: a lane's 32 bytes of floats are two copies, and the second finds its sectors there.
// Around L1 the float32 step took 160 instead of 123 us for 47 million weights.)
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async8(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 shared16(uint32_t at) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(at));
  return r;
}
__device__ __forceinline__ uint2 shared8(uint32_t at) {
  uint2 r;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(r.x), "=r"(r.y) : "r"(at));
  return r;
}

// One block of a warp in shared memory: parameters (or masters), gradients, codes of both moments,
// each lane's 16 (8) bytes beside its neighbour's.
template <typename P, typename G, bool MASTER>
struct Stage8 {
  using W = typename std::conditional<MASTER, float, P>::type;
  static constexpr int kG = kStateBlock * (int)sizeof(W), kM = kG + kStateBlock * (int)sizeof(G), kV = kM + kStateBlock;
  static constexpr int kBytes = kV + kStateBlock;
  __device__ static void fetch(uint32_t at, const Tensor8<P, G>& t, long long first, int lane) {
    const W* p;
    if constexpr (MASTER) p = t.w + first;
    else p = t.p + first;
#pragma unroll
    for (int k = 0; k < (int)sizeof(W) / 2; ++k) copy_async16(at + k * 512 + lane * 16, reinterpret_cast<const uint4*>(p) + k);
#pragma unroll
    for (int k = 0; k < (int)sizeof(G) / 2; ++k)
      copy_async16(at + kG + k * 512 + lane * 16, reinterpret_cast<const uint4*>(t.g + first) + k);
    copy_async8(at + kM + lane * 8, t.m + first);
    copy_async8(at + kV + lane * 8, t.v + first);
  }
};
constexpr int kStages8 = 3;
template <typename P, typename G, bool MASTER>
constexpr int kShared8 = kWarps * kStages8 * Stage8<P, G, MASTER>::kBytes;

// A warp takes `per_warp` consecutive blocks (at most 32: a lane holds the scales of one). Each lane copies its
// share of a block to shared memory kStages8 - 1 blocks ahead, asynchronously, and later reads back what it
// copied itself, so no barrier is needed and the loads in flight hold no registers. Scales are read and
// written once per task, lane k's for block k.
// 436M bf16 weights: 655 us, 6.7 TB/s (1592 with plain loads, 1039 with the next block's loads in
// registers); under the power cap, at 1.58 GHz, 755 us: 41 instructions an element keep the ALU pipe busy.
// Lists that are not aligned (8 parameters, 8 gradients and 8 masters each on a boundary of their size, 32 bytes
// with float32) go element by element (ragged_block8): 100M weights 306 us with bf16 parameters and 405 with
// float32, 3.3 and 4.0 TB/s, where aligned ones take 156 and 246.
template <typename P, typename G, bool MASTER, int CAP>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm8)
adamw8_kernel(const __grid_constant__ AdamW8Args<CAP> a) {
  using Stage = Stage8<P, G, MASTER>;
  extern __shared__ __align__(16) unsigned char ring[];
  float f;
  if (!read_factor(a.c.grad_scale, f)) return;
  const int block = from_the_end();
  const int e = find_tensor(a.start, a.c.count, block);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Tensor8<P, G> t = {static_cast<P*>(a.p[e]), a.w[e], static_cast<const G*>(a.g[e]), a.m[e], a.v[e], a.ms[e],
                           a.vs[e], a.numel[e], a.step[e], a.rs[e], a.key[e]};
  const AdamWConsts c = a.c;
  const long long blocks = (t.numel + kStateBlock - 1) / kStateBlock;
  const long long whole = a.vec_ok[e] ? t.numel / kStateBlock : 0;  // blocks that the vector path takes
  const long long b0 = ((long long)(block - a.start[e]) * kWarps + warp) * a.per_warp;
  const int n = (int)min(max(whole - b0, 0ll), (long long)a.per_warp);
  const uint32_t slots = smem_u32(ring) + warp * kStages8 * Stage::kBytes;
  const long long first = b0 * kStateBlock + lane * 8;
#pragma unroll
  for (int k = 0; k < kStages8 - 1; ++k) {
    if (k < n) Stage::fetch(slots + k * Stage::kBytes, t, first + k * kStateBlock, lane);
    copy_async_commit();
  }
  float ms = 0.f, vs = 0.f, m_top = 0.f, v_top = 0.f;  // of block `lane` of the task
  if (lane < n) {
    ms = t.ms[b0 + lane];
    vs = t.vs[b0 + lane];
  }
  int slot = 0, ahead = kStages8 - 1;
  for (int k = 0; k < n; ++k) {
    if (k + kStages8 - 1 < n)
      Stage::fetch(slots + ahead * Stage::kBytes, t, first + (k + kStages8 - 1) * kStateBlock, lane);
    copy_async_commit();
    ahead = ahead + 1 == kStages8 ? 0 : ahead + 1;
    copy_async_wait<kStages8 - 1>();
    const uint32_t at = slots + slot * Stage::kBytes;
    slot = slot + 1 == kStages8 ? 0 : slot + 1;
    float2 pj[4], gj[4], mj[4], vj[4];
    Raw<typename Stage::W, 8> rp;
    Raw<G, 8> rg;
#pragma unroll
    for (int h = 0; h < rp.kWords; ++h) rp.w[h] = shared16(at + h * 512 + lane * 16);
#pragma unroll
    for (int h = 0; h < rg.kWords; ++h) rg.w[h] = shared16(at + Stage::kG + h * 512 + lane * 16);
    rp.unpack(pj);
    rg.unpack(gj);
    decode8<STATE_EXP_AVG>(shared8(at + Stage::kM + lane * 8), __shfl_sync(0xffffffffu, ms, k), mj);
    decode8<STATE_EXP_AVG_SQ>(shared8(at + Stage::kV + lane * 8), __shfl_sync(0xffffffffu, vs, k), vj);
    step8(c, t, f, pj, gj, mj, vj);
    const long long i = first + k * kStateBlock;
    Raw<P, 8> out;
    out.pack(pj);
    out.template store<true>(t.p + i);
    if constexpr (MASTER) {
      rp.pack(pj);
      rp.template store<true>(t.w + i);
    }
    const float m_amax = warp_max(amax_bits(mj)), v_amax = warp_max(amax_bits_unsigned(vj));
    if (lane == k) {
      m_top = m_amax;
      v_top = v_amax;
    }
    uint32_t r[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t bits = random_word((uint32_t)(i >> 2) + h, t.key);
#pragma unroll
      for (int j = 0; j < 4; ++j) r[4 * h + j] = random_bits(bits, j);
    }
    float m_inv, v_inv;
    both_factors(m_amax, v_amax, lane, m_inv, v_inv);
    __stcs(reinterpret_cast<uint2*>(t.m + i), encode8<STATE_EXP_AVG>(mj, m_inv, r));
    __stcs(reinterpret_cast<uint2*>(t.v + i), encode8<STATE_EXP_AVG_SQ>(vj, v_inv, r));
  }
  if (lane < n) {
    t.ms[b0 + lane] = block_scale<STATE_EXP_AVG>(m_top);
    t.vs[b0 + lane] = block_scale<STATE_EXP_AVG_SQ>(v_top);
  }
  const long long end = min(blocks, b0 + a.per_warp);
  for (long long b = b0 + n; b < end; ++b) ragged_block8<P, G, MASTER>(c, t, f, b);
}

// ---------------------------------------------------------------------------
// Conversion of moments: 32-bit (or 16-bit) values <-> codes and scales. Bound by HBM: 218M values from float32
// 155 us (7.05 TB/s), to bf16 98 us (6.7 TB/s). Where values (by 8) or codes are not aligned, elements go one by one: 100M
// values from float32 101 to 109 us (75 aligned), from bf16 107 to 115 (55); back, where values and codes are never aligned
// together, to float32 164 us (77) and to bf16 151 (48).
// ---------------------------------------------------------------------------
constexpr int kBlocksPerWarp = 4;
constexpr int kBlocksPerChunk = kWarps * kBlocksPerWarp;

template <int CAP>
struct ConvertArgs {
  void* x[CAP];
  uint8_t* codes[CAP];
  float* scales[CAP];
  long long numel[CAP];
  int start[CAP + 1];
  unsigned char head[CAP];  // first element aligned in both lists (quantize: 0), or kNoHead
  int count;
  uint32_t half;  // half a code (2^19), added before the cut: to nearest
};

template <typename T, int KIND, int CAP>
__global__ void __launch_bounds__(kThreads)
quantize_kernel(const __grid_constant__ ConvertArgs<CAP> a) {
  const int t = find_tensor(a.start, a.count, (int)blockIdx.x);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long numel = a.numel[t];
  const long long blocks = (numel + kStateBlock - 1) / kStateBlock;
  const T* x = static_cast<const T*>(a.x[t]);
  uint8_t* codes = a.codes[t];
  const long long first = (long long)((int)blockIdx.x - a.start[t]) * kBlocksPerChunk + warp;
  // Half a code is added before the cut. It is an argument because of the compiler (nvcc 12.9.86): with the
  // constant 1 << 19 in its place the first element of every pair came out as 255 in this kernel, while the
  // same expression in a kernel of its own is right for all 2^32 bit patterns, with either. The tests compare
  // every code with the format's definition.
  const uint32_t r[8] = {a.half, a.half, a.half, a.half, a.half, a.half, a.half, a.half};
#pragma unroll
  for (int k = 0; k < kBlocksPerWarp; ++k) {
    const long long b = first + (long long)k * kWarps;
    if (b >= blocks) return;
    const long long base = b * kStateBlock;
    const long long at = base + lane * 8;
    const bool vec = a.head[t] == 0 && base + kStateBlock <= numel;
    float2 xj[4];
    if (vec) {
      Raw<T, 8> rx;
      rx.load(x + at);
      rx.unpack(xj);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const long long i = base + lane + 32 * j;
        (j & 1 ? xj[j / 2].y : xj[j / 2].x) = i < numel ? to_float<T>(x[i]) : 0.f;
      }
    }
    const float amax = warp_max(amax_bits(xj)), inv = block_factor<KIND>(amax);
    if (lane == 0) a.scales[t][b] = block_scale<KIND>(amax);
    const uint2 c = encode8<KIND, true>(xj, inv, r);
    if (vec) {
      __stcs(reinterpret_cast<uint2*>(codes + at), c);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const long long i = base + lane + 32 * j;
        if (i < numel) codes[i] = byte_of(c, j);
      }
    }
  }
}

// A warp expands 1024 consecutive elements, 16 codes a lane at a time, so that codes are read and values
// written 16 bytes and more to a lane. It starts where codes and values are both aligned; 16 codes from
// there may lie in two blocks.
template <typename T, int KIND, int CAP>
__global__ void __launch_bounds__(kThreads)
dequantize_kernel(const __grid_constant__ ConvertArgs<CAP> a) {
  constexpr int kPieces = kBlocksPerWarp / 2, kSpan = kBlocksPerWarp * kStateBlock;
  const int t = find_tensor(a.start, a.count, (int)blockIdx.x);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long numel = a.numel[t];
  T* x = static_cast<T*>(a.x[t]);
  const uint8_t* codes = a.codes[t];
  const float* scales = a.scales[t];
  const bool vec = a.head[t] != kNoHead;
  const int head = vec ? a.head[t] : 0;
  const long long task = (long long)((int)blockIdx.x - a.start[t]) * kWarps + warp, base = task * kSpan + head;
  const auto single = [&](long long i) { x[i] = from_float<T>(decode1<KIND>(codes[i], scales[i / kStateBlock])); };
  if (task == 0 && lane < head) single(lane);
  if (base >= numel) return;
  if (!vec) {
    const int n = (int)min(numel - base, (long long)kSpan);
#pragma unroll 8
    for (int i = lane; i < n; i += 32) single(base + i);
    return;
  }
  uint4 c[kPieces];
  float first[kPieces], second[kPieces];
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long at = base + 512 * k + 16 * lane;
    if (at + 16 <= numel) {
      c[k] = __ldcs(reinterpret_cast<const uint4*>(codes + at));
      first[k] = scales[at / kStateBlock];
      second[k] = scales[(at + 15) / kStateBlock];
    }
  }
#pragma unroll
  for (int k = 0; k < kPieces; ++k) {
    const long long at = base + 512 * k + 16 * lane;
    if (at + 16 <= numel) {
      const int split = kStateBlock - (int)(at % kStateBlock);  // elements before the second block
      float2 lo[4], hi[4], all[8];
      decode8<KIND>(make_uint2(c[k].x, c[k].y), lo);
      decode8<KIND>(make_uint2(c[k].z, c[k].w), hi);
      if (split >= 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) all[j] = mul2(j < 4 ? lo[j & 3] : hi[j & 3], both(first[k]));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          all[j] = mul2(j < 4 ? lo[j & 3] : hi[j & 3], make_float2(2 * j < split ? first[k] : second[k],
                                                                 2 * j + 1 < split ? first[k] : second[k]));
      }
      Raw<T, 16> rx;
      rx.pack(all);
      rx.store(x + at);
    } else {
      for (long long i = at; i < numel; ++i) single(i);
    }
  }
}

// ---------------------------------------------------------------------------
// Global gradient norm. Squares are added in float32 over the 8 or 16 elements of a 32-byte access and in
// float64 from there on, in an order that depends on sizes, alignment and the device alone. Where these squares overflow,
// or are so small that they lose bits, they are taken in float64 instead: the norm is right over the
// whole range of the type. Bound by HBM: 437 MB 65 us (6.7 TB/s).
// ---------------------------------------------------------------------------
template <int CAP>
struct NormArgs {
  void* x[CAP];
  long long numel[CAP];
  int start[CAP + 1];
  unsigned char dtype[CAP];
  unsigned char head[CAP];  // elements before the first that is aligned
  int count, chunks;
  double* partials;
};

// A thread takes 32 bytes at a time, kNormIters times in a chunk.
constexpr int kNormIters = 4;
constexpr int kNormBlocksPerSm = 4;
template <typename T>
constexpr int kNormVec = 32 / (int)sizeof(T);
template <typename T>
constexpr int kNormChunk = kThreads * kNormIters * kNormVec<T>;

template <int N>
__device__ __forceinline__ double squares(const float (&x)[N]) {
  float s[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < N; ++j) s[j & 1] = fmaf(x[j], x[j], s[j & 1]);
  const float sum = s[0] + s[1];
  if (sum < 3e38f && sum > 1e-30f) return (double)sum;
  uint32_t any = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) any |= __float_as_uint(x[j]) << 1;
  if (any == 0) return 0.0;
  double d = 0.0;
#pragma unroll
  for (int j = 0; j < N; ++j) d += (double)x[j] * (double)x[j];
  return d;
}

// A chunk of a tensor: `head` elements behind the tensor's start, of which the first chunk also takes the head.
template <typename T>
__device__ __forceinline__ double chunk_squares(const T* x, int chunk, int head, long long numel) {
  constexpr int V = kNormVec<T>, kChunk = kNormChunk<T>;
  double acc = 0.0;
  const long long base = (long long)chunk * kChunk + head;
  const int end = (int)min(numel - base, (long long)kChunk), done = end / V * V;
  x += base;
  if (end == kChunk) {
    Raw<T, V> rx[kNormIters];  // all loads before the sums, whose rare branch they could not cross
#pragma unroll
    for (int k = 0; k < kNormIters; ++k) rx[k].load(x + (k * kThreads + threadIdx.x) * V);
#pragma unroll
    for (int k = 0; k < kNormIters; ++k) {
      float v[V];
      rx[k].unpack(v);
      acc += squares(v);
    }
  } else {
    for (int i = threadIdx.x * V; i < done; i += kThreads * V) {
      Raw<T, V> rx;
      rx.load(x + i);
      float v[V];
      rx.unpack(v);
      acc += squares(v);
    }
  }
  int i = done + threadIdx.x;  // fewer than V behind the last whole piece, and the head
  if (i >= end) i = chunk == 0 && (int)threadIdx.x >= kThreads - head ? (int)threadIdx.x - kThreads : end;
  if (i < end) {
    const double v = (double)to_float<T>(x[i]);
    acc += v * v;
  }
  return acc;
}

// Sum over the block, to every thread; the order of the additions is fixed.
__device__ __forceinline__ double block_sum(double v, double (&warps)[kWarps]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int k = 0; k < kWarps; ++k) s += warps[k];
  return s;
}

template <int CAP>
__device__ __forceinline__ double squares_of(const NormArgs<CAP>& a, int chunk) {
  const int t = find_tensor(a.start, a.count, chunk);
  const int k = chunk - a.start[t], head = a.head[t];
  const long long n = a.numel[t];
  if (a.dtype[t] == DT_F32) return chunk_squares(static_cast<const float*>(a.x[t]), k, head, n);
  if (a.dtype[t] == DT_BF16) return chunk_squares(static_cast<const __nv_bfloat16*>(a.x[t]), k, head, n);
  return chunk_squares(static_cast<const __half*>(a.x[t]), k, head, n);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads, kNormBlocksPerSm)
norm_partial_kernel(const __grid_constant__ NormArgs<CAP> a) {
  __shared__ double warps[kWarps];
  griddep_launch_dependents();
  double acc = 0.0;
  for (int chunk = blockIdx.x; chunk < a.chunks; chunk += gridDim.x) acc += squares_of(a, chunk);
  acc = block_sum(acc, warps);
  if (threadIdx.x == 0) a.partials[blockIdx.x] = acc;
}

// {norm, factor that clips}; a NaN stays.
__device__ __forceinline__ float2 norm_and_factor(double sum, float max_norm) {
  const float norm = (float)sqrt(sum), q = max_norm / (norm + 1e-6f);
  return make_float2(norm, q > 1.f ? 1.f : q);
}
// The factor that grad_norm hands out: none where the norm is not finite.
__device__ __forceinline__ float handed_out(float2 r) {
  return fabsf(r.x) <= 3.402823466e38f ? r.y : __int_as_float(0x7fffffff);
}

// From the partial sums: every block that needs the result adds them up in the same order.
__device__ __forceinline__ float2 finish_norm(const double* partials, int n, float max_norm, double (&warps)[kWarps]) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) acc += partials[i];
  return norm_and_factor(block_sum(acc, warps), max_norm);
}

__global__ void __launch_bounds__(kThreads)
norm_finish_kernel(const double* partials, int n, float max_norm, float* out2) {
  __shared__ double warps[kWarps];
  griddep_launch_dependents();
  griddep_wait();
  const float2 r = finish_norm(partials, n, max_norm, warps);
  if (threadIdx.x == 0) {
    out2[0] = r.x;
    out2[1] = handed_out(r);
  }
}

template <typename T>
__device__ __forceinline__ void scale_chunk(T* x, int chunk, int head, long long numel, float f) {
  constexpr int V = kNormVec<T>, kChunk = kNormChunk<T>;
  const long long base = (long long)chunk * kChunk + head;
  const int end = (int)min(numel - base, (long long)kChunk), done = end / V * V;
  x += base;
#pragma unroll 2
  for (int i = threadIdx.x * V; i < done; i += kThreads * V) {
    Raw<T, V> rx;
    rx.load(x + i);
    float v[V];
    rx.unpack(v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= f;
    rx.pack(v);
    rx.store(x + i);
  }
  int i = done + threadIdx.x;
  if (i >= end) i = chunk == 0 && (int)threadIdx.x >= kThreads - head ? (int)threadIdx.x - kThreads : end;
  if (i < end) x[i] = from_float<T>(to_float<T>(x[i]) * f);
}

template <int CAP>
__device__ __forceinline__ void scale_one(const NormArgs<CAP>& a, int chunk, float f) {
  const int t = find_tensor(a.start, a.count, chunk);
  const int k = chunk - a.start[t], head = a.head[t];
  const long long n = a.numel[t];
  if (a.dtype[t] == DT_F32) scale_chunk(static_cast<float*>(a.x[t]), k, head, n, f);
  else if (a.dtype[t] == DT_BF16) scale_chunk(static_cast<__nv_bfloat16*>(a.x[t]), k, head, n, f);
  else scale_chunk(static_cast<__half*>(a.x[t]), k, head, n, f);
}

template <int CAP>
__global__ void __launch_bounds__(kThreads)
clip_kernel(const __grid_constant__ NormArgs<CAP> a, int partials, float max_norm, float* out2) {
  __shared__ double warps[kWarps];
  const float2 r = finish_norm(a.partials, partials, max_norm, warps);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    out2[0] = r.x;
    out2[1] = r.y;
  }
  if (r.y == 1.f) return;  // nothing to clip: x * 1 is x
  // from the end: what the norm's pass read last is still in L2 (189 MB: 92 -> 78 us with the norm, 437 MB: 221 -> 208)
  for (int chunk = a.chunks - 1 - (int)blockIdx.x; chunk >= 0; chunk -= gridDim.x) scale_one(a, chunk, r.y);
}

// The whole of a call with few chunks in one launch of one cluster: the blocks' sums meet in shared memory
// instead of global memory, and each block scales what it summed. For 25 vectors of 768 a call returns after
// 7.6 instead of 10.5 us (a launch less), while the device takes 4.0 instead of 3.1 us.
constexpr int kClusterBlocks = 8, kClusterChunks = 32;

template <int CAP, bool CLIP>
__global__ void __cluster_dims__(kClusterBlocks) __launch_bounds__(kThreads)
norm_cluster_kernel(const __grid_constant__ NormArgs<CAP> a, float max_norm, float* out2) {
  namespace cg = cooperative_groups;
  __shared__ double warps[kWarps];
  __shared__ double mine;
  const cg::cluster_group cluster = cg::this_cluster();
  griddep_launch_dependents();
  double acc = 0.0;
  for (int chunk = blockIdx.x; chunk < a.chunks; chunk += kClusterBlocks) acc += squares_of(a, chunk);
  acc = block_sum(acc, warps);
  if (threadIdx.x == 0) mine = acc;
  cluster.sync();
  double sum = 0.0;
#pragma unroll
  for (int k = 0; k < kClusterBlocks; ++k) sum += *cluster.map_shared_rank(&mine, k);
  cluster.sync();  // no block leaves while its sum is read
  const float2 r = norm_and_factor(sum, max_norm);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    out2[0] = r.x;
    out2[1] = CLIP ? r.y : handed_out(r);
  }
  if constexpr (CLIP) {
    if (r.y == 1.f) return;
    for (int chunk = blockIdx.x; chunk < a.chunks; chunk += kClusterBlocks) scale_one(a, chunk, r.y);
  }
}

// ---------------------------------------------------------------------------
// Host side: tables are filled tensor by tensor and launched when full.
// ---------------------------------------------------------------------------
inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline int elem_bytes(int dtype) { return dtype == DT_F32 ? 4 : 2; }

struct BiasCorrection {  // lr / (1 - b1^t) and 1 / sqrt(1 - b2^t); most tensors of a call share t
  int64_t t = 0;
  float step = 0.f, rs = 0.f;
  void set(const AdamWCall& c, int64_t now) {
    if (now == t) return;
    t = now;
    step = (float)(c.lr / (1.0 - std::pow(c.beta1, (double)t)));
    rs = (float)(1.0 / std::sqrt(1.0 - std::pow(c.beta2, (double)t)));
  }
};

struct ListStart {
  const void* p;
  size_t bytes;  // of an element
};
// The first element, under N, at which all lists are aligned to N elements; kNoHead: there is none.
template <int N>
int common_head(std::initializer_list<ListStart> lists) {
  uintptr_t off = 0;  // (a null pointer is aligned)
  for (const ListStart& l : lists) off |= reinterpret_cast<uintptr_t>(l.p) & (N * l.bytes - 1);
  if (off == 0) return 0;
  int head = -1;
  for (const ListStart& l : lists) {
    if (!l.p) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(l.p) / l.bytes;  // (aligned to its elements)
    const int h = (int)((N - at % N) % N);
    if (head >= 0 && h != head) return kNoHead;
    head = h;
  }
  return head;
}

// Launches a kernel that waits for its predecessor on the stream by itself (griddep_wait): its launch, with
// arguments of up to 32 KB, then runs beside the predecessor's end where that one allows it
// (griddep_launch_dependents). A norm's two kernels and a step with its factor follow one another so: 63.4 ->
// 59.6 us for norm and step of 150 packed float16 tensors. Not the clipping pass: its blocks, which share the
// work out evenly, were placed unevenly as the norm's left (437 MB: 121 -> 129 us).
template <typename... Params, typename... Args>
int launch_after(void (*kernel)(Params...), int grid, size_t shared, cudaStream_t stream, bool dependent,
                 const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent && dependent_launch_enabled() ? 1 : 0;
  MB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
  MB_CUDA_CHECK(cudaGetLastError());
  return OK;
}

// Adds `chunks` to the running total of a launch; false when the launch must go out first.
inline bool fits(int total, int64_t chunks) { return chunks <= (int64_t)INT32_MAX - total; }

template <typename P, typename G, bool MASTER, int CAP>
int adamw32_launch(const AdamWCall& c, const AdamWConsts& consts, cudaStream_t stream) {
  AdamW32Args<CAP> a;
  a.c = consts;
  BiasCorrection bias;
  const double bytes = (MASTER ? sizeof(P) + 8.0 : 2.0 * sizeof(P)) + sizeof(G) + 16.0;
  int n = 0;
  double elems = 0;
  a.start[0] = 0;
  for (int i = 0; i <= c.count; ++i) {
    constexpr int V = kVec32<P>;
    int head = 0;
    int64_t chunks = 0;
    if (i < c.count && c.numel[i] > 0) {
      head = common_head<V>({{c.param[i], sizeof(P)}, {c.grad[i], sizeof(G)}, {c.exp_avg[i], 4}, {c.exp_avg_sq[i], 4},
                             {MASTER ? c.master[i] : nullptr, 4}});
      if (head >= c.numel[i]) head = kNoHead;
      chunks = (c.numel[i] - (head == kNoHead ? 0 : head) + kChunk32<P> - 1) / kChunk32<P>;
    }
    if (i == c.count || n == CAP || !fits(a.start[n], chunks)) {
      if (n > 0) {
        a.c.count = n;
        LaunchScope scope(K_ADAMW, elems * bytes, stream);
        const int rc = launch_after(adamw32_kernel<P, G, MASTER, CAP>, a.start[n], 0, stream, c.grad_scale != nullptr, a);
        if (rc != OK) return rc;
      }
      n = 0;
      elems = 0;
    }
    if (chunks == 0) continue;
    a.p[n] = c.param[i];
    a.w[n] = MASTER ? static_cast<float*>(c.master[i]) : nullptr;
    a.g[n] = c.grad[i];
    a.m[n] = static_cast<float*>(c.exp_avg[i]);
    a.v[n] = static_cast<float*>(c.exp_avg_sq[i]);
    a.numel[n] = c.numel[i];
    bias.set(c, c.steps[i]);
    a.step[n] = bias.step;
    a.rs[n] = bias.rs;
    a.head[n] = (unsigned char)head;
    a.start[n + 1] = a.start[n] + (int)chunks;
    elems += (double)c.numel[i];
    ++n;
  }
  return OK;
}

// Blocks per warp: long tasks keep the pipeline of copies full, short ones leave a shorter tail. As many as
// make one round of resident warps, at most kMostPerWarp: two layers of 436M bf16 weights take 877, 723,
// 677, 658, 664, 679 us with 2, 4, 6, 8, 12, 16 blocks a warp, 150 tensors of 72 thousand float32
// weights 38 us with one and 28 with eight, 90 of 53 thousand 16.6 with one, 12.4 with six, 15.1 with eight.
constexpr int kMostPerWarp = 8;
inline int blocks_per_warp(double blocks, int sms) {
  const int per = (int)std::ceil(blocks / ((double)sms * kBlocksPerSm8 * kWarps));
  return per < 1 ? 1 : per > kMostPerWarp ? kMostPerWarp : per;
}

template <typename P, typename G, bool MASTER, int CAP>
int adamw8_launch(const AdamWCall& c, const AdamWConsts& consts, cudaStream_t stream) {
  AdamW8Args<CAP> a;
  a.c = consts;
  BiasCorrection bias;
  const double bytes = (MASTER ? sizeof(P) + 8.0 : 2.0 * sizeof(P)) + sizeof(G) + 4.0 + 16.0 / kStateBlock;
  constexpr int kShared = kShared8<P, G, MASTER>;
  if (kShared > 48 * 1024)
    MB_CUDA_CHECK(cudaFuncSetAttribute(adamw8_kernel<P, G, MASTER, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, kShared));
  int sms = 0, rc = device_sm_count(&sms);
  if (rc != OK) return rc;
  double blocks = 0;
  for (int i = 0; i < c.count; ++i) blocks += (double)(c.numel[i] / kStateBlock + 1);
  a.per_warp = blocks_per_warp(blocks, sms);
  int n = 0;
  double elems = 0;
  a.start[0] = 0;
  for (int i = 0; i <= c.count; ++i) {
    const int64_t per = (int64_t)kWarps * a.per_warp * kStateBlock;
    const int64_t chunks = i < c.count ? (c.numel[i] + per - 1) / per : 0;
    if (i == c.count || n == CAP || !fits(a.start[n], chunks)) {
      if (n > 0) {
        a.c.count = n;
        LaunchScope scope(K_ADAMW, elems * bytes, stream);
        rc = launch_after(adamw8_kernel<P, G, MASTER, CAP>, a.start[n], kShared, stream, c.grad_scale != nullptr, a);
        if (rc != OK) return rc;
      }
      n = 0;
      elems = 0;
    }
    if (chunks == 0) continue;
    a.p[n] = c.param[i];
    a.w[n] = MASTER ? static_cast<float*>(c.master[i]) : nullptr;
    a.g[n] = c.grad[i];
    a.m[n] = static_cast<uint8_t*>(c.exp_avg[i]);
    a.ms[n] = static_cast<float*>(c.exp_avg_scale[i]);
    a.v[n] = static_cast<uint8_t*>(c.exp_avg_sq[i]);
    a.vs[n] = static_cast<float*>(c.exp_avg_sq_scale[i]);
    a.numel[n] = c.numel[i];
    bias.set(c, c.steps[i]);
    a.step[n] = bias.step;
    a.rs[n] = bias.rs;
    a.key[n] = random_key(c.seed, c.steps[i]);
    a.vec_ok[n] = aligned(a.p[n], 8 * sizeof(P)) && aligned(a.g[n], 8 * sizeof(G)) && aligned(a.m[n], 8) &&
                  aligned(a.v[n], 8) && aligned(a.w[n], 32);
    a.start[n + 1] = a.start[n] + (int)chunks;
    elems += (double)c.numel[i];
    ++n;
  }
  return OK;
}

// Tensors per launch. Up to 32764 bytes of arguments hold several hundred, but handing them over takes the
// host about 1 us for 6 KB: calls with fewer tensors take a smaller table. A call on 128 tensors of 768 elements
// takes 14.3 us (AdamW), 12.8 (norm) and 15.7 (clipping) with the table for 160, and 17.8, 15.1 and 20.0 with the
// largest one; from 160 to 161 tensors it gets 2, 2 and 3.5 us longer. With 320 in the place of 160, 161 / 200 / 300
// tensors took 0.6 / 3.3 / 1.6 us less (AdamW), 1.5 / 1.2 / 0.2 (norm) and 1.3 / 2.8 / 2.0 (clipping), and 90 and 150
// tensors 0.4 to 7 us more.
constexpr int kCapFew = 64, kCapSome = 160, kCapAdamW32 = 512, kCapAdamW8 = 384, kCapConvert = 512, kCapNorm = 1024;

// f(std::integral_constant<int, CAP>) with the table that fits `count` tensors.
template <int MOST, typename F>
int with_table(int count, F f) {
  if (count <= kCapFew) return f(std::integral_constant<int, kCapFew>());
  if (count <= kCapSome) return f(std::integral_constant<int, kCapSome>());
  return f(std::integral_constant<int, MOST>());
}

template <typename P, typename G, bool MASTER>
int adamw_launch(const AdamWCall& c, const AdamWConsts& consts, cudaStream_t stream) {
  if (c.exp_avg_scale)
    return with_table<kCapAdamW8>(
        c.count, [&](auto cap) { return adamw8_launch<P, G, MASTER, decltype(cap)::value>(c, consts, stream); });
  return with_table<kCapAdamW32>(
      c.count, [&](auto cap) { return adamw32_launch<P, G, MASTER, decltype(cap)::value>(c, consts, stream); });
}

template <typename P, typename G>
int adamw_launch(const AdamWCall& c, const AdamWConsts& consts, cudaStream_t stream) {
  if constexpr (sizeof(P) == 4) return adamw_launch<P, G, false>(c, consts, stream);
  else return c.master ? adamw_launch<P, G, true>(c, consts, stream) : adamw_launch<P, G, false>(c, consts, stream);
}

template <int CAP, typename LAUNCH>
int for_each_norm_table(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double* partials,
                        LAUNCH launch) {
  NormArgs<CAP> a;
  a.partials = partials;
  int n = 0;
  double bytes = 0;
  a.start[0] = 0;
  for (int i = 0; i <= count; ++i) {
    int head = 0;
    int64_t chunks = 0;
    if (i < count && numel[i] > 0) {
      const int size = elem_bytes(dtypes[i]), chunk = size == 4 ? kNormChunk<float> : kNormChunk<__half>;
      head = (int)((32 - reinterpret_cast<uintptr_t>(tensors[i]) % 32) % 32) / size;
      if (head > numel[i]) head = (int)numel[i];
      chunks = numel[i] == head ? 1 : (numel[i] - head + chunk - 1) / chunk;
    }
    if (i == count || n == CAP || !fits(a.start[n], chunks)) {
      if (n > 0) {
        a.count = n;
        a.chunks = a.start[n];
        const int rc = launch(a, bytes);
        if (rc != OK) return rc;
      }
      n = 0;
      bytes = 0;
    }
    if (chunks == 0) continue;
    a.x[n] = tensors[i];
    a.numel[n] = numel[i];
    a.dtype[n] = (unsigned char)dtypes[i];
    a.head[n] = (unsigned char)head;
    a.start[n + 1] = a.start[n] + (int)chunks;
    bytes += (double)numel[i] * elem_bytes(dtypes[i]);
    ++n;
  }
  return OK;
}

constexpr int kNormTables = 64;  // launches of the norm kernel per call: 64 * 1024 tensors

int norm_grid(int chunks, int* grid) {
  int sms = 0;
  const int rc = device_sm_count(&sms);
  if (rc != OK) return rc;
  *grid = chunks < sms * kNormBlocksPerSm ? chunks : sms * kNormBlocksPerSm;
  return OK;
}

template <int CAP>
int norm_partials(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double* partials,
                  int* n_partials, cudaStream_t stream) {
  int used = 0, tables = 0;
  const int rc = for_each_norm_table<CAP>(
      tensors, numel, dtypes, count, partials, [&](NormArgs<CAP>& a, double bytes) -> int {
        int grid = 0;
        const int rc = norm_grid(a.chunks, &grid);
        if (rc != OK) return rc;
        if (++tables > kNormTables) return set_error(ERR_UNSUPPORTED, "gradient norm: too many tensors in one call");
        a.partials = partials + used;
        LaunchScope scope(K_GRAD_NORM, bytes, stream);
        norm_partial_kernel<CAP><<<grid, kThreads, 0, stream>>>(a);
        MB_CUDA_CHECK(cudaGetLastError());
        used += grid;
        return OK;
      });
  *n_partials = used;
  return rc;
}

template <typename T, int KIND, bool TO_CODES, int CAP>
int convert_launch(void* const* x, void* const* codes, void* const* scales, const int64_t* numel, int count,
                   cudaStream_t stream) {
  ConvertArgs<CAP> a;
  a.half = 1u << 19;
  int n = 0;
  double elems = 0;
  a.start[0] = 0;
  for (int i = 0; i <= count; ++i) {
    const int64_t per = (int64_t)kBlocksPerChunk * kStateBlock;
    int head = 0;
    int64_t chunks = 0;
    if (i < count && numel[i] > 0) {
      if (TO_CODES) {  // (its blocks start at the tensor's first element)
        head = aligned(x[i], 8 * sizeof(T)) && aligned(codes[i], 8) ? 0 : kNoHead;
      } else {
        head = common_head<16>({{x[i], sizeof(T)}, {codes[i], 1}});
        if (head > numel[i]) head = kNoHead;
      }
      chunks = (numel[i] + per - 1) / per;  // (a head only makes the last chunk shorter)
    }
    if (i == count || n == CAP || !fits(a.start[n], chunks)) {
      if (n > 0) {
        a.count = n;
        LaunchScope scope(K_STATE_CONVERT, elems * (sizeof(T) + 1.0 + 4.0 / kStateBlock), stream);
        if (TO_CODES) quantize_kernel<T, KIND, CAP><<<a.start[n], kThreads, 0, stream>>>(a);
        else dequantize_kernel<T, KIND, CAP><<<a.start[n], kThreads, 0, stream>>>(a);
        MB_CUDA_CHECK(cudaGetLastError());
      }
      n = 0;
      elems = 0;
    }
    if (chunks == 0) continue;
    a.x[n] = x[i];
    a.codes[n] = static_cast<uint8_t*>(codes[i]);
    a.scales[n] = static_cast<float*>(scales[i]);
    a.numel[n] = numel[i];
    a.head[n] = (unsigned char)head;
    a.start[n + 1] = a.start[n] + (int)chunks;
    elems += (double)numel[i];
    ++n;
  }
  return OK;
}

template <bool TO_CODES>
int convert(void* const* x, void* const* codes, void* const* scales, const int64_t* numel, int count, int dtype,
            int kind, cudaStream_t stream) {
  return with_table<kCapConvert>(count, [&](auto cap) {
    constexpr int CAP = decltype(cap)::value;
    const bool avg = kind == STATE_EXP_AVG;
#define MB_CONVERT(T)                                                                                      \
  (avg ? convert_launch<T, STATE_EXP_AVG, TO_CODES, CAP>(x, codes, scales, numel, count, stream)           \
       : convert_launch<T, STATE_EXP_AVG_SQ, TO_CODES, CAP>(x, codes, scales, numel, count, stream))
    return dtype == DT_F32 ? MB_CONVERT(float) : dtype == DT_BF16 ? MB_CONVERT(__nv_bfloat16) : MB_CONVERT(__half);
#undef MB_CONVERT
  });
}

}  // namespace

int run_adamw(const AdamWCall& c, cudaStream_t stream) {
  AdamWConsts k;
  k.b1 = (float)c.beta1;
  k.w1 = (float)(1.0 - c.beta1);
  k.b2 = (float)c.beta2;
  k.w2 = (float)(1.0 - c.beta2);
  k.eps = (float)c.eps;
  k.decay = (float)(1.0 - c.lr * c.weight_decay);
  k.one = 1.f;
  k.grad_scale = c.grad_scale;
  k.count = 0;
  const bool wide = c.grad_dtype == DT_F32;
  if (c.param_dtype == DT_F32) return adamw_launch<float, float>(c, k, stream);
  if (c.param_dtype == DT_BF16)
    return wide ? adamw_launch<__nv_bfloat16, float>(c, k, stream) : adamw_launch<__nv_bfloat16, __nv_bfloat16>(c, k, stream);
  return wide ? adamw_launch<__half, float>(c, k, stream) : adamw_launch<__half, __half>(c, k, stream);
}

int grad_norm_partials(int* n) {
  int sms = 0;
  const int rc = device_sm_count(&sms);
  *n = sms * kNormBlocksPerSm * kNormTables;
  return rc;
}

namespace {
// A call with few chunks as one launch. False: it has more (or none), and nothing was launched.
template <bool CLIP>
int norm_in_one_launch(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double max_norm,
                       float* out2, cudaStream_t stream, bool* done) {
  *done = false;
  if (count > kCapFew) return OK;
  return for_each_norm_table<kCapFew>(
      tensors, numel, dtypes, count, nullptr, [&](NormArgs<kCapFew>& a, double bytes) -> int {
        int sms = 0;
        const int rc = device_sm_count(&sms);
        if (rc != OK || a.chunks > kClusterChunks) return rc;
        *done = true;  // (the lists of up to kCapFew tensors with so few chunks are one table)
        LaunchScope scope(K_GRAD_NORM, CLIP ? 3.0 * bytes : bytes, stream);
        norm_cluster_kernel<kCapFew, CLIP><<<kClusterBlocks, kThreads, 0, stream>>>(a, (float)max_norm, out2);
        MB_CUDA_CHECK(cudaGetLastError());
        return OK;
      });
}

template <int CAP>
int clip_launch(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double max_norm,
                float* out2, double* partials, cudaStream_t stream) {
  int n = 0, launched = 0;
  int rc = norm_partials<CAP>(tensors, numel, dtypes, count, partials, &n, stream);
  if (rc != OK) return rc;
  rc = for_each_norm_table<CAP>(
      tensors, numel, dtypes, count, partials, [&](NormArgs<CAP>& a, double bytes) -> int {
        int grid = 0;
        const int rc = norm_grid(a.chunks, &grid);
        if (rc != OK) return rc;
        ++launched;
        LaunchScope scope(K_GRAD_NORM, 2.0 * bytes, stream);
        clip_kernel<CAP><<<grid, kThreads, 0, stream>>>(a, n, (float)max_norm, out2);
        MB_CUDA_CHECK(cudaGetLastError());
        return OK;
      });
  if (rc != OK || launched) return rc;
  LaunchScope scope(K_GRAD_NORM, 0.0, stream);  // nothing but empty tensors: the norm is 0
  return launch_after(norm_finish_kernel, 1, 0, stream, false, static_cast<const double*>(partials), 0, (float)max_norm, out2);
}
}  // namespace

int run_grad_norm(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double max_norm,
                  float* out2, double* partials, cudaStream_t stream) {
  bool done = false;
  int n = 0, rc = norm_in_one_launch<false>(tensors, numel, dtypes, count, max_norm, out2, stream, &done);
  if (rc != OK || done) return rc;
  rc = with_table<kCapNorm>(count, [&](auto cap) {
    return norm_partials<decltype(cap)::value>(tensors, numel, dtypes, count, partials, &n, stream);
  });
  if (rc != OK) return rc;
  LaunchScope scope(K_GRAD_NORM, 8.0 * n, stream);
  return launch_after(norm_finish_kernel, 1, 0, stream, n > 0, static_cast<const double*>(partials), n, (float)max_norm, out2);
}

int run_clip(void* const* tensors, const int64_t* numel, const int* dtypes, int count, double max_norm,
             float* out2, double* partials, cudaStream_t stream) {
  bool done = false;
  const int rc = norm_in_one_launch<true>(tensors, numel, dtypes, count, max_norm, out2, stream, &done);
  if (rc != OK || done) return rc;
  return with_table<kCapNorm>(count, [&](auto cap) {
    return clip_launch<decltype(cap)::value>(tensors, numel, dtypes, count, max_norm, out2, partials, stream);
  });
}

int run_quantize(void* const* src, void* const* codes, void* const* scales, const int64_t* numel, int count,
                 int dtype, int kind, cudaStream_t stream) {
  return convert<true>(src, codes, scales, numel, count, dtype, kind, stream);
}

int run_dequantize(void* const* codes, void* const* scales, void* const* dst, const int64_t* numel, int count,
                   int dtype, int kind, cudaStream_t stream) {
  return convert<false>(dst, codes, scales, numel, count, dtype, kind, stream);
}

}  // namespace mb
