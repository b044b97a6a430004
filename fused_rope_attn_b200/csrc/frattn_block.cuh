// Device helpers shared by the transformer-block operators (layer norm, linear
// layer with epilogue, 8-bit activation checkpoints): vector access to rows of
// any alignment, the checkpoint format, and the activations with derivatives.
#pragma once
#include "frattn_kernel.cuh"

namespace frattn {

// ---------------------------------------------------------------- rows as vectors
// VEC consecutive elements of a row. A kernel instance for VEC is launched only
// when every row start is aligned to min(16, VEC * sizeof(T)) bytes and VEC
// divides the row length (row_vec below), so no access leaves its row.
template <typename T>
__device__ __forceinline__ float elem_f32(T x);
template <>
__device__ __forceinline__ float elem_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float elem_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float elem_f32<__half>(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T f32_elem(float x);
template <>
__device__ __forceinline__ float f32_elem<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 f32_elem<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half f32_elem<__half>(float x) { return __float2half_rn(x); }

template <int BYTES>
struct RawVec;
template <>
struct RawVec<1> { using type = uint8_t; };
template <>
struct RawVec<2> { using type = uint16_t; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<16> { using type = uint4; };

__device__ __forceinline__ void raw_words(uint16_t r, uint32_t* w) { w[0] = r; }
__device__ __forceinline__ void raw_words(uint8_t r, uint32_t* w) { w[0] = r; }
__device__ __forceinline__ void raw_words(uint32_t r, uint32_t* w) { w[0] = r; }
__device__ __forceinline__ void raw_words(uint2 r, uint32_t* w) { w[0] = r.x; w[1] = r.y; }
__device__ __forceinline__ void raw_words(uint4 r, uint32_t* w) { w[0] = r.x; w[1] = r.y; w[2] = r.z; w[3] = r.w; }

// VEC elements as 32-bit words, as loaded (loads of several vectors can be in flight
// before any of them is converted; element-sized pieces would each take a register).
template <typename T, int VEC>
struct Vec {
  static constexpr int kBytes = VEC * static_cast<int>(sizeof(T));
  static constexpr int kPart = kBytes > 16 ? 16 : kBytes;
  static constexpr int kParts = kBytes / kPart;
  static constexpr int kPartWords = kPart < 4 ? 1 : kPart / 4;
  using Raw = typename RawVec<kPart>::type;
  uint32_t w[kParts * kPartWords];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) raw_words(__ldcg(reinterpret_cast<const Raw*>(p) + i), w + i * kPartWords);
  }
  __device__ __forceinline__ void get(float (&v)[VEC]) const {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const __half2 h = *reinterpret_cast<const __half2*>(&w[i / 2]);
        v[i] = i & 1 ? __high2float(h) : __low2float(h);
      }
    }
  }
  // v rounded to T, to p
  static __device__ __forceinline__ void put(T* p, const float (&v)[VEC]) {
    if constexpr (std::is_same<T, float>::value) {
      if constexpr (VEC == 1) p[0] = v[0];
      else if constexpr (VEC == 2) *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
      else
#pragma unroll
        for (int i = 0; i < VEC / 4; ++i)
          reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else if constexpr (VEC == 1) {
      p[0] = f32_elem<T>(v[0]);
    } else if constexpr (VEC == 2) {
      *reinterpret_cast<uint32_t*>(p) = pack2<T>(v[0], v[1]);
    } else if constexpr (VEC == 4) {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    } else {
      *reinterpret_cast<uint4*>(p) =
          make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  }
};

// VEC int8 codes of a checkpoint, as loaded.
template <int VEC>
struct CodeVec {
  static constexpr int kWords = VEC < 4 ? 1 : VEC / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const int8_t* p) {
    raw_words(__ldcg(reinterpret_cast<const typename RawVec<VEC>::type*>(p)), w);
  }
  __device__ __forceinline__ void get(float step, float (&v)[VEC]) const {
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = static_cast<float>(static_cast<int8_t>(w[i / 4] >> (8 * (i & 3)))) * step;
  }
};

// Largest vector width of {8, 4, 2, 1} elements of esz bytes that every listed
// pointer and row stride (elements) allows for rows of C elements.
struct RowVec {
  int C, esz;
  int v = 8;
  RowVec(int C_, int esz_) : C(C_), esz(esz_) {
    while (C % v) v /= 2;
  }
  RowVec& row(const void* p, long long stride, int e = 0) {
    if (!p) return *this;
    const int es = e ? e : esz;
    auto ok = [&](int w) {
      const int a = w * es < 16 ? w * es : 16;
      return reinterpret_cast<uintptr_t>(p) % a == 0 && (stride * es) % a == 0;
    };
    while (v > 1 && !ok(v)) v /= 2;
    return *this;
  }
};

// Launch whose start overlaps the end of the kernel before it in the stream (programmatic
// dependent launch): the block operators are short, and follow each other. Every kernel
// launched this way executes griddep_wait() before its first access to global memory: it
// waits until the kernels before have completed and their writes are visible to it, to
// plain loads too. None of its loads is read-only by declaration (__ldg, const __restrict__),
// which would let the non-coherent path serve it with lines older than the writes waited
// for. Most go past L1 (ld.global.cg, asynchronous copies), since they are read once;
// the bias, the residual, misaligned parameters and rows of more than 8192 columns are
// plain loads. griddep_launch_dependents() comes once a kernel has nothing left to set up;
// one that does not call it (layer_norm_bwd_kernel) lets the next start when it ends.
template <typename... P, typename... A>
inline int launch_overlapped(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, A... args) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = grid;
  lc.blockDim = block;
  lc.dynamicSmemBytes = smem;
  lc.stream = st;
  lc.attrs = attr;
  lc.numAttrs = cluster > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&lc, kern, static_cast<P>(args)...);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? 0 : FRATTN_E_CUDA;
}

inline bool aligned_to(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// ---------------------------------------------------------------- 8-bit checkpoints
// A row of C values in blocks of 32: codes [T, 32 nb] int8, scale bytes [T, nb],
// nb = ceil(C / 32). With amax = f 2^q, 1/2 <= f < 1, the block's largest
// magnitude: e = max(q - 7, -126), scale byte e + 127, code = rint(x / 2^e)
// limited to [-127, 127]. A power-of-two scale makes both directions exact but
// for that one rounding: x 2^-e is exact in 32 bits, and code 2^e has 7
// significant bits, so it is exact in bf16 and fp32 (and, for values that came
// from fp16, in fp16): a gradient computed from a checkpoint rounds it no
// further. A block that holds an infinity or a NaN gets scale byte 255 and
// stands for NaN throughout, so that it is not lost.
constexpr int kPackBlock = 32;
constexpr uint32_t kPackNan = 255;

__host__ __device__ inline long long pack_blocks(int C) { return (static_cast<long long>(C) + kPackBlock - 1) / kPackBlock; }

// Scale byte of a block from the largest (x as bits) & 0x7fffffff of its values
// (integer order of the magnitudes; NaNs come out on top).
__device__ __forceinline__ uint32_t pack_scale(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;  // q + 126
  return e == 255u ? kPackNan : (e > 7u ? e : 7u) - 6u;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// 2^-e of a scale byte; 0 for a NaN block (whose codes are then 0).
__device__ __forceinline__ float pack_inv(uint32_t scale) {
  return scale == kPackNan ? 0.f : __uint_as_float((254u - scale) << 23);
}
// 2^e of a scale byte; NaN for a NaN block.
__device__ __forceinline__ float pack_step(uint32_t scale) {
  return scale == kPackNan ? __uint_as_float(0x7fffffffu) : __uint_as_float(scale << 23);
}
// Largest magnitude that a code of the block stands for; 0 for a NaN block, whose
// codes are 0.
__device__ __forceinline__ float pack_limit(uint32_t scale) {
  return scale == kPackNan ? 0.f : 127.f * __uint_as_float(scale << 23);
}
// Code of x in the low byte: x / 2^e is exact, and adding 1.5 2^23 rounds it to the
// nearest integer (ties to even) in two's complement.
__device__ __forceinline__ uint32_t pack_code(float x, float inv, float lim) {
  return __float_as_uint(fmaf(fminf(fmaxf(x, -lim), lim), inv, 12582912.f));
}
__device__ __forceinline__ uint32_t pack_code4(float a, float b, float c, float d, float inv, float lim) {
  const uint32_t lo = __byte_perm(pack_code(a, inv, lim), pack_code(b, inv, lim), 0x0040);
  const uint32_t hi = __byte_perm(pack_code(c, inv, lim), pack_code(d, inv, lim), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}

// max(m, |a|, |b|); a NaN among them stays.
__device__ __forceinline__ float max3_abs(float m, float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}
// Codes of N values (four to a word) of a block with largest magnitude m and scale byte
// sc. Two values at a time on the packed fp32 pipe; the limit to 127 steps, which only a
// block whose largest magnitude is within 2^-7 of a power of two needs, is a branch.
template <int N>
__device__ __forceinline__ void pack_codes(const float (&v)[N], float m, uint32_t sc, uint32_t (&codes)[N / 4]) {
  const float inv = pack_inv(sc);
  if (fabsf(m) * inv < 127.5f) {  // (false for a NaN block: NaN, or infinity x 0)
    const uint64_t inv2 = f2pack(inv, inv), magic = f2pack(12582912.f, 12582912.f);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      float a, b, c, d;
      f2unpack(fma2(f2pack(v[4 * i], v[4 * i + 1]), inv2, magic), a, b);
      f2unpack(fma2(f2pack(v[4 * i + 2], v[4 * i + 3]), inv2, magic), c, d);
      const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
      codes[i] = __byte_perm(lo, hi, 0x5410);
    }
  } else {
    const float lim = pack_limit(sc);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) codes[i] = pack_code4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv, lim);
  }
}
// A whole block of 32 held by one thread: its codes and scale byte.
__device__ __forceinline__ uint32_t pack32(const float (&v)[32], uint32_t (&codes)[8]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < 32; i += 2) m = max3_abs(m, v[i], v[i + 1]);
  const uint32_t sc = pack_scale(abs_bits(m));
  pack_codes<32>(v, m, sc, codes);
  return sc;
}

// ---------------------------------------------------------------- activations
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return f2pack(x, x); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The standard normal distribution function in the form of Hastings (Abramowitz and
// Stegun, Handbook of Mathematical Functions, 7.1.26): for z <= 0
//   e^(-z^2 / 2) (a1 t + ... + a6 t^6), t = 1 / (1 + p |z|),
// and 1 minus that at -z for z > 0. p and a were fitted here, by a linear programme over
// z in [-14.5, 0] (where e^(-z^2 / 2) leaves 32 bits), to the smallest relative error under
// an absolute one of 1.2e-7: 2^-14.8 of the function's value, a fifth of an fp16 rounding,
// since gelu of a negative value is z times just this tail. (The five terms of 7.1.26 are
// fitted to the absolute error alone: 5e-4 of the value at z = -4, 7e-3 at -7, more than a
// bf16 rounding.) A third of erff's instructions and no branch; the sixth term takes 1 %
// (9216 x 1280 -> 3424 with gelu 74.5 -> 75.3 us, its backward pass 172.7 -> 174.5).

// Two values at a time: the polynomial parts on the packed fp32 pipe, and one reciprocal
// for both (1 / a = b / (a b)): the special-function unit, a quarter as wide as the
// others, otherwise sets the pace (derivative of gelu_tanh over 9216 x 3424: 17 us of
// 47). Arguments are limited so that the product stays finite, at magnitudes where the
// distribution function or the sigmoid is 0 or 1 to 2^-58; the limit also turns a NaN
// into a number, so that it comes back through the factor z alone and does not reach its
// neighbour. A sigmoid below that is 0, not 2^-58, where z multiplies it
// (sigmoid_factor): z itself is not limited, and has 2^127 in bf16.
__device__ __forceinline__ uint64_t rcp_pair(float a, float b) {
  const float r = rcp_fast(a * b);
  return f2pack(r * b, r * a);
}
__device__ __forceinline__ float limit_f(float x, float lim) { return fminf(fmaxf(x, -lim), lim); }
// 1 / (1 + 2^u) of two u, each at most 60
__device__ __forceinline__ uint64_t sigmoid_pair(float u0, float u1) {
  float a, b;
  f2unpack(add2(f2pack(exp2_fast(u0), exp2_fast(u1)), both(1.f)), a, b);
  return rcp_pair(a, b);
}
// normal_cdf of two values, and e^(-z^2 / 2)
__device__ __forceinline__ void normal_cdf_pair(float a, float b, float& c0, float& c1, uint64_t& e) {
  const float za = limit_f(a, 64.f), zb = limit_f(b, 64.f);
  float t0, t1, e0, e1, q0, q1;
  f2unpack(fma2(f2pack(fabsf(za), fabsf(zb)), both(0.295f), both(1.f)), t0, t1);
  const uint64_t t = rcp_pair(t0, t1), z = f2pack(za, zb);
  f2unpack(mul2(mul2(z, both(-0.7213475204444817f)), z), e0, e1);
  e = f2pack(exp2_fast(e0), exp2_fast(e1));
  uint64_t q = fma2(t, both(-0.08374395332f), both(0.2509855948f));
  q = fma2(q, t, both(-0.05372828448f));
  q = fma2(q, t, both(0.1601948595f));
  q = fma2(q, t, both(0.1079014198f));
  q = fma2(q, t, both(0.1183903083f));
  f2unpack(mul2(mul2(q, t), e), q0, q1);
  c0 = za < 0.f ? q0 : 1.f - q0;
  c1 = zb < 0.f ? q1 : 1.f - q1;
}
// gelu_tanh's sigmoid: 1 / (1 + e^-2u), u = sqrt(2 / pi) (z + 0.044715 z^3), |z| <= 7.4
__device__ __forceinline__ uint64_t tanh_pair(uint64_t z, uint64_t z2) {
  float u0, u1;
  f2unpack(mul2(fma2(z2, both(-0.10294324f), both(-2.3022082f)), z), u0, u1);
  return sigmoid_pair(u0, u1);
}
constexpr float kTanhLimit = 7.4f, kSiluLimit = 41.f;  // 2^u <= 2^60
// The sigmoid s of a z limited to [-lim, lim] as the factor of z (a NaN z keeps s)
__device__ __forceinline__ float sigmoid_factor(float z, float s, float lim) { return z < -lim ? 0.f : s; }

template <int ACT>
__device__ __forceinline__ void act_f2(float& a, float& b) {
  if constexpr (ACT == FRATTN_ACT_GELU) {
    float c0, c1;
    uint64_t e;
    normal_cdf_pair(a, b, c0, c1, e);
    a *= c0;
    b *= c1;
  } else if constexpr (ACT == FRATTN_ACT_GELU_TANH) {
    const uint64_t z = f2pack(limit_f(a, kTanhLimit), limit_f(b, kTanhLimit));
    float s0, s1;
    f2unpack(tanh_pair(z, mul2(z, z)), s0, s1);
    a *= sigmoid_factor(a, s0, kTanhLimit);
    b *= sigmoid_factor(b, s1, kTanhLimit);
  } else if constexpr (ACT == FRATTN_ACT_SILU) {
    float u0, u1;
    f2unpack(mul2(f2pack(limit_f(a, kSiluLimit), limit_f(b, kSiluLimit)), both(-1.4426950408889634f)), u0, u1);
    f2unpack(sigmoid_pair(u0, u1), u0, u1);
    a *= sigmoid_factor(a, u0, kSiluLimit);
    b *= sigmoid_factor(b, u1, kSiluLimit);
  } else if constexpr (ACT == FRATTN_ACT_RELU) {
    a = a > 0.f ? a : (a != a ? a : 0.f);
    b = b > 0.f ? b : (b != b ? b : 0.f);
  }
}

// Derivatives of two values at a time, times d0 and d1.
template <int ACT>
__device__ __forceinline__ void act_grad_f2(float a, float b, float& d0, float& d1) {
  float g0, g1;
  if constexpr (ACT == FRATTN_ACT_GELU) {
    uint64_t e;
    normal_cdf_pair(a, b, g0, g1, e);
    const uint64_t z = f2pack(limit_f(a, 64.f), limit_f(b, 64.f));
    f2unpack(fma2(mul2(z, e), both(0.3989422804014327f), f2pack(g0, g1)), g0, g1);
  } else if constexpr (ACT == FRATTN_ACT_GELU_TANH) {
    const uint64_t z = f2pack(limit_f(a, kTanhLimit), limit_f(b, kTanhLimit)), z2 = mul2(z, z), s = tanh_pair(z, z2);
    const uint64_t w = mul2(mul2(s, z), add2(both(1.f), mul2(s, both(-1.f))));
    f2unpack(fma2(w, fma2(z2, both(0.21406445f), both(1.5957691f)), s), g0, g1);
  } else if constexpr (ACT == FRATTN_ACT_SILU) {
    const uint64_t z = f2pack(limit_f(a, kSiluLimit), limit_f(b, kSiluLimit));
    float u0, u1;
    f2unpack(mul2(z, both(-1.4426950408889634f)), u0, u1);
    const uint64_t s = sigmoid_pair(u0, u1);
    f2unpack(fma2(mul2(s, z), add2(both(1.f), mul2(s, both(-1.f))), s), g0, g1);
  } else if constexpr (ACT == FRATTN_ACT_RELU) {
    g0 = a > 0.f ? 1.f : 0.f;
    g1 = b > 0.f ? 1.f : 0.f;
  } else {
    g0 = g1 = 1.f;
  }
  d0 *= a == a ? g0 : a;
  d1 *= b == b ? g1 : b;
}

}  // namespace frattn
