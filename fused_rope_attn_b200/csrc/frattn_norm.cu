// Layer norm forward and backward, and 8-bit activation checkpoints (sm_100a).
//
// Forward, per row of C values:
//   mean = sum x / C, rstd = 1 / sqrt(sum (x - mean)^2 / C + eps),
//   y = (x - mean) rstd w + b
// Backward, with h = (x - mean) rstd and g = dy w:
//   dx = rstd (g - mean(g) - h mean(g h)),  dw = sum over rows of dy h,
//   db = sum over rows of dy
// All sums are kept in 32 bits; the variance is the sum of squared differences
// from the mean over values held in registers (no difference of large sums).
//
// Both are bound by the bytes of the rows. A team of 1 to 8 warps works on a row at a
// time, up to 40 columns to a lane held in registers, so that a row is read from memory
// once (fewer columns and more warps cost more instructions per value than the memory
// leaves time for: with 8 columns to a lane a value took 28 instructions). Teams are
// persistent: their rows come through a ring in shared memory of the team's own, filled
// by asynchronous 16-byte copies, which hold no registers and, being cut at 16-byte
// boundaries of the address and not of the row, take rows of any alignment. With few
// rows a block of more warps takes each, straight from memory. The weight gradients stay
// in the registers of the lane that owns the column; at the end the teams of a block add
// theirs through shared memory, each block writes one partial row, and column_finish
// adds the partial rows, all in a fixed order (no atomics: the same bits every run).
//
// Measured, bf16: forward 32768 x 1280 in 29.0 us (5.8 TB/s, 0.88 of the copy rate),
// 9216 x 1280 in 10.9 us; backward 53.6 us (4.7 TB/s) and 24.3 us, of which starting,
// joining the gradients and adding the partial rows take 10. The backward's inner loop
// is bound by instruction issue and shared-memory reads rather than by memory.
#include "frattn_block.cuh"
#include "frattn_row_pieces.h"

namespace frattn {

struct NormParams {
  const void* x;        // [T, C] rows of x_stride elements (null: codes / scales)
  long long x_stride;
  const int8_t* codes;  // [T, 32 nb]
  const uint8_t* scales;  // [T, nb]
  const void* w;        // [C] or null (ones)
  const void* b;        // [C] or null (zeros), forward only
  int w_f32;            // w, b, dw, db are fp32 (else the element type)
  int w_vec;            // w and b are 16-byte aligned (forward)
  const void* dy;       // [T, C] rows of dy_stride elements, backward only
  long long dy_stride;
  void* out;            // y or dx
  long long out_stride;
  float* mean;          // [T] written by the forward (or null), read by the backward
  float* rstd;
  float* partial;       // [blocks][2][C] (backward)
  int T, C;
  float eps;
};

namespace {

// Sum over the block's threads (wide rows); every thread gets it. `red` must not be
// reused before the next barrier but one.
template <int R>
__device__ __forceinline__ void block_sum(float (&s)[R], float* red) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
  }
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) red[warp * R + r] = s[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) s[r] = 0.f;
  for (int w = 0; w < nw; ++w) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] += red[w * R + r];
  }
}

__device__ __forceinline__ float param_at(const void* p, int f32, int dtype_bf16, int c, float fill) {
  if (!p) return fill;
  if (f32) return __ldcg(static_cast<const float*>(p) + c);
  return dtype_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[c]) : __half2float(static_cast<const __half*>(p)[c]);
}

// ---------------------------------------------------------------- row ring
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, uint32_t bytes) {
  // reads `bytes` (<= 16) of the 16, the rest of dst is zeros; dst and src 16-byte aligned
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Bytes of ring for a row of up to `bytes` bytes at any alignment: the 16-byte pieces of
// memory that it touches (the row starts address mod 16 bytes into them) and a piece of
// zeros. Slots are zero from the row's end on to start with and every copy ends in a
// piece of zeros, so what lies between a row and the last column its team covers is zero
// always.
__host__ __device__ inline int row_slot(int bytes) { return (bytes + 15) / 16 * 16 + 32; }

__device__ __forceinline__ uint32_t lead(const uint8_t* row) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row)) & 15u;
}

// A team's threads (t of n) copy the row at `row` into the slot dst; nothing before
// `base`, the matrix's first row, is read, nor past the row's end.
__device__ __forceinline__ void fetch_row(const uint8_t* row, int bytes, const uint8_t* base, uint8_t* dst, int t, int n) {
  const int off = static_cast<int>(lead(row));
  const uint8_t* src = row - off;
  if (t == 0 && src < base) {
    for (int i = off; i < 16 && i < off + bytes; ++i) dst[i] = src[i];
    t += n;
  }
  const uint32_t to = smem_u32(dst);
  row_pieces(off, bytes, t, n, [&](int at, int from, int size) { copy16_async(to + at, src + from, size); });
}

// The team: `warps` warps of the block with a named barrier of their own.
struct Team {
  int id, t, n;  // team of the block, thread of the team, threads of a team
  __device__ __forceinline__ explicit Team(int warps) {
    n = 32 * warps;
    id = threadIdx.x / n;
    t = threadIdx.x - id * n;
  }
  __device__ __forceinline__ void sync() const {
    if (n == 32) __syncwarp();
    else named_bar_sync(1 + id, n);
  }
  // Sums of R values over the team. `red` (8 R floats of the team's) is free again after
  // the team's next sync.
  template <int R>
  __device__ __forceinline__ void sum(float (&s)[R], float* red) const {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
    if (n == 32) return;
    if ((t & 31) == 0) {
#pragma unroll
      for (int r = 0; r < R; ++r) red[(t >> 5) * R + r] = s[r];
    }
    sync();
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = 0.f;
    for (int w = 0; w < n / 32; ++w) {
#pragma unroll
      for (int r = 0; r < R; ++r) s[r] += red[w * R + r];
    }
  }
};

// Zeros in a row's slot from the row's end on.
__device__ __forceinline__ void clear_tail(uint8_t* slot, int bytes, int slot_bytes, const Team& team) {
  for (int at = bytes / 16 * 16 + 16 * team.t; at < slot_bytes; at += 16 * team.n)
    *reinterpret_cast<uint4*>(slot + at) = make_uint4(0, 0, 0, 0);
}

// A lane's columns: 8 NU of them in units of 8, each unit 8 / VEC vectors of VEC. A warp's
// columns are consecutive, 256 to a unit; vectors lie 32 VEC columns apart, which makes
// their addresses one register and constants.
template <int VEC, int NU>
__device__ __forceinline__ int lane_col(const Team& team) {
  return (team.t >> 5) * (NU * 256) + (team.t & 31) * VEC;
}
template <int VEC>
__device__ __forceinline__ int unit_col(int c0, int u, int j) {  // first column of vector j of unit u
  return c0 + (u * (8 / VEC) + j) * 32 * VEC;
}

// Units of a warp whose 256 columns all exist (they need no comparisons).
template <int NU>
__device__ __forceinline__ int full_units(const Team& team, int C) {
  const int n = (C - (team.t >> 5) * (NU * 256)) / 256;
  return n < 0 ? 0 : n;
}

// Eight values of unit u: f(c, v) loads the vector at column c into v.
template <int VEC, typename F>
__device__ __forceinline__ void unit_load(int c0, int u, float (&v)[8], F&& f) {
#pragma unroll
  for (int j = 0; j < 8 / VEC; ++j) {
    float x[VEC];
    f(unit_col<VEC>(c0, u, j), x);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[j * VEC + e] = x[e];
  }
}
// From a row in shared memory.
template <typename T, int VEC>
__device__ __forceinline__ void unit_get(const uint8_t* row, int c0, int u, float (&v)[8]) {
  unit_load<VEC>(c0, u, v, [&](int c, float (&x)[VEC]) {
    Vec<T, VEC> r;
#pragma unroll
    for (int i = 0; i < Vec<T, VEC>::kParts; ++i)
      raw_words(reinterpret_cast<const typename Vec<T, VEC>::Raw*>(row + c * sizeof(T))[i], r.w + i * Vec<T, VEC>::kPartWords);
    r.get(x);
  });
}
// From a checkpoint's row in shared memory: codes and scale bytes.
template <int VEC>
__device__ __forceinline__ void unit_get_packed(const uint8_t* codes, const uint8_t* scales, int c0, int u, float (&v)[8]) {
  unit_load<VEC>(c0, u, v, [&](int c, float (&x)[VEC]) {
    CodeVec<VEC> q;
    raw_words(*reinterpret_cast<const typename RawVec<VEC>::type*>(codes + c), q.w);
    q.get(pack_step(scales[c / kPackBlock]), x);
  });
}
// Eight values of unit u to a row of T in global memory.
template <typename T, int VEC>
__device__ __forceinline__ void unit_put(T* row, int c0, int u, int full, int C, const float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 8 / VEC; ++j) {
    const int c = unit_col<VEC>(c0, u, j);
    float f[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) f[e] = v[j * VEC + e];
    if (u < full || c < C) Vec<T, VEC>::put(row + c, f);
  }
}

// Weights in shared memory in 32 bits, C rounded up to 8 of them (zeros there). For
// vectors of 8 the two float4 of a vector lie half the array apart, so that the lanes'
// reads have no bank conflicts.
template <int VEC>
__device__ __forceinline__ int param_slot(int c, int C8) {
  return VEC == 8 ? ((c >> 2) & 1) * (C8 / 2) + (c >> 3) * 4 + (c & 3) : c;
}
template <int VEC>
__device__ __forceinline__ void unit_param(const float* w, int c0, int u, int C8, float (&v)[8]) {
  unit_load<VEC>(c0, u, v, [&](int c, float (&x)[VEC]) {
    if constexpr (VEC == 1) {
      x[0] = w[c];
    } else {
      const float4 a = *reinterpret_cast<const float4*>(w + (VEC == 8 ? c / 2 : c));
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
      if constexpr (VEC == 8) {
        const float4 b = *reinterpret_cast<const float4*>(w + C8 / 2 + c / 2);
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
      }
    }
  });
}

// The block copies a parameter vector there: eight values to a thread and step, whose
// loads are in flight together (a block may be a single warp).
template <typename T, int VEC>
__device__ __forceinline__ void stage_param(float* to, const void* src, int f32, float fill, int C, int C8) {
  const bool vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
#pragma unroll 4
  for (int c = 8 * static_cast<int>(threadIdx.x); c < C8; c += 8 * static_cast<int>(blockDim.x)) {
    float v[8];
    if (!src) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = fill;
    } else if (vec && c + 8 <= C) {
      if (f32) {
        Vec<float, 8> x;
        x.load(static_cast<const float*>(src) + c);
        x.get(v);
      } else {
        Vec<T, 8> x;
        x.load(static_cast<const T*>(src) + c);
        x.get(v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = c + e < C ? c + e : C - 1;  // (past C: any value, the gradient there is 0)
        v[e] = f32 ? __ldcg(static_cast<const float*>(src) + at) : elem_f32<T>(static_cast<const T*>(src)[at]);
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
      *reinterpret_cast<float4*>(to + param_slot<VEC>(c + 4 * h, C8)) =
          make_float4(v[4 * h], v[4 * h + 1], v[4 * h + 2], v[4 * h + 3]);
  }
}

// Rows of a team's ring: one worked on, one on its way (a third measured no faster: the
// SM's other teams have theirs on their way too).
constexpr int kPasses = 2;

// How a block's shared memory is laid out: parameters, then per team the ring and the
// reduction's floats.
struct NormLayout {
  int warps;   // of a team
  int teams;   // of a block
  int slot;    // ring bytes of a row
  int cols;                // columns that a team covers, C or more: what the rows and parameters are padded to
  int params, team_bytes;  // bytes
};

// Parameters of unit u from global memory (every row reads them: they stay in L1).
template <typename T, int VEC>
__device__ __forceinline__ void unit_param_global(const void* p, int f32, int vec, float fill, int c0, int u, int C,
                                                  float (&v)[8]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fill;
  } else if (f32) {
    unit_load<VEC>(c0, u, v, [&](int c, float (&x)[VEC]) {
      const float* src = static_cast<const float*>(p) + c;
      Vec<float, VEC> r;  // (past C: whatever is there, for no output)
      if (vec) {
        if (c < C) r.load(src);
        r.get(x);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = c < C ? __ldcg(src + e) : 0.f;
      }
    });
  } else {
    unit_load<VEC>(c0, u, v, [&](int c, float (&x)[VEC]) {
      const T* src = static_cast<const T*>(p) + c;
      Vec<T, VEC> r;
      if (vec) {
        if (c < C) r.load(src);
        r.get(x);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = c < C ? elem_f32<T>(src[e]) : 0.f;
      }
    });
  }
}

// Few rows: a block per row.
template <typename T, int VEC, int NU>
__global__ void __launch_bounds__(256) layer_norm_fwd_few_kernel(const NormParams p) {
  __shared__ float red[1][2][8];
  const Team team(blockDim.x / 32);
  const long long row = blockIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  const int c0 = lane_col<VEC, NU>(team), full = full_units<NU>(team, p.C);
  const T* src = static_cast<const T*>(p.x) + row * p.x_stride;
  float x[NU][8], s[1] = {0.f};
#pragma unroll
  for (int u = 0; u < NU; ++u)
    unit_load<VEC>(c0, u, x[u], [&](int c, float (&v)[VEC]) {
      Vec<T, VEC> r;
#pragma unroll
      for (int i = 0; i < Vec<T, VEC>::kParts * Vec<T, VEC>::kPartWords; ++i) r.w[i] = 0;
      if (c < p.C) r.load(src + c);
      r.get(v);
    });
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += x[u][e];
  team.sum(s, red[team.id][0]);
  const float inv_c = 1.f / static_cast<float>(p.C), mean = s[0] * inv_c;
  s[0] = 0.f;
#pragma unroll
  for (int u = 0; u < NU; ++u) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[u][e] -= mean;
    if (u >= full) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (unit_col<VEC>(c0, u, e / VEC) >= p.C) x[u][e] = 0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) s[0] += x[u][e] * x[u][e];
  }
  team.sum(s, red[team.id][1]);
  const float rstd = rsqrtf(s[0] * inv_c + p.eps);
  if (team.t == 0) {
    if (p.mean) p.mean[row] = mean;
    if (p.rstd) p.rstd[row] = rstd;
  }
  T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
  for (int u = 0; u < NU; ++u) {
    float g[8], h[8];
    unit_param_global<T, VEC>(p.w, p.w_f32, p.w_vec, 1.f, c0, u, p.C, g);
    unit_param_global<T, VEC>(p.b, p.w_f32, p.w_vec, 0.f, c0, u, p.C, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[u][e] = x[u][e] * rstd * g[e] + h[e];
    unit_put<T, VEC>(out, c0, u, full, p.C, x[u]);
  }
}

// Many rows: persistent teams whose rows come through the ring.
template <typename T, int VEC, int NU>
__global__ void __launch_bounds__(256, NU > 3 ? 3 : 4) layer_norm_fwd_kernel(const NormParams p, const NormLayout l) {
  extern __shared__ __align__(16) uint8_t smem[];
  float* w = reinterpret_cast<float*>(smem);
  float* b = w + l.cols;
  const Team team(l.warps);
  const int c0 = lane_col<VEC, NU>(team), full = full_units<NU>(team, p.C);
  uint8_t* ring = smem + l.params + team.id * l.team_bytes;
  float* red = reinterpret_cast<float*>(ring + l.team_bytes) - 16;  // the last 64 bytes of the team's part
  constexpr int kT = static_cast<int>(sizeof(T));
  const uint8_t* const base = static_cast<const uint8_t*>(p.x);
  const long long stride = p.x_stride * kT;
  const int step = gridDim.x * l.teams, bytes = p.C * kT, first = blockIdx.x * l.teams + team.id;
  long long fetched = first;
  int into = 0;
  auto fetch = [&] {
    if (fetched < p.T) fetch_row(base + fetched * stride, bytes, base, ring + into * l.slot, team.t, team.n);
    copies_commit();
    fetched += step;
    into = into + 1 == kPasses ? 0 : into + 1;
  };
  for (int k = 0; k < kPasses; ++k) clear_tail(ring + k * l.slot, bytes, l.slot, team);
  team.sync();
  griddep_wait();
  griddep_launch_dependents();
  for (int k = 0; k < kPasses - 1; ++k) fetch();
  stage_param<T, VEC>(w, p.w, p.w_f32, 1.f, p.C, l.cols);
  stage_param<T, VEC>(b, p.b, p.w_f32, 0.f, p.C, l.cols);
  __syncthreads();
  const float inv_c = 1.f / static_cast<float>(p.C);
  int at = 0;
  for (long long row = first; row < p.T; row += step) {
    copies_wait<kPasses - 2>();
    team.sync();  // the row is in the ring, and nobody reads the one before it any more
    fetch();
    const uint8_t* src = ring + at * l.slot + lead(base + row * stride);
    float x[NU][8], s[1] = {0.f};
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      unit_get<T, VEC>(src, c0, u, x[u]);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += x[u][e];
    }
    team.sum(s, red);
    const float mean = s[0] * inv_c;
    s[0] = 0.f;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u][e] -= mean;
      if (u >= full) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (unit_col<VEC>(c0, u, e / VEC) >= p.C) x[u][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) s[0] += x[u][e] * x[u][e];
    }
    team.sum(s, red + 8);
    const float rstd = rsqrtf(s[0] * inv_c + p.eps);
    if (team.t == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      float g[8], h[8];
      unit_param<VEC>(w, c0, u, l.cols, g);
      unit_param<VEC>(b, c0, u, l.cols, h);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[u][e] = x[u][e] * rstd * g[e] + h[e];
      unit_put<T, VEC>(out, c0, u, full, p.C, x[u]);
    }
    at = at + 1 == kPasses ? 0 : at + 1;
  }
}

// Rows of more than 8192 columns: one block per row, the row is read three times
// (from L2 after the first).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_fwd_wide_kernel(const NormParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  __shared__ float red[2][32];
  const float inv_c = 1.f / static_cast<float>(p.C);
  for (long long row = blockIdx.x; row < p.T; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) s[0] += elem_f32<T>(x[c]);
    block_sum<1>(s, red[0]);
    const float mean = s[0] * inv_c;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      const float d = elem_f32<T>(x[c]) - mean;
      s[0] += d * d;
    }
    block_sum<1>(s, red[1]);
    const float rstd = rsqrtf(s[0] * inv_c + p.eps);
    if (threadIdx.x == 0) {
      if (p.mean) p.mean[row] = mean;
      if (p.rstd) p.rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      const float w = param_at(p.w, p.w_f32, kBf16, c, 1.f), b = param_at(p.b, p.w_f32, kBf16, c, 0.f);
      out[c] = f32_elem<T>((elem_f32<T>(x[c]) - mean) * rstd * w + b);
    }
  }
}

template <typename T, int VEC, int NU, bool PACKED>
__global__ void __launch_bounds__(384) layer_norm_bwd_kernel(const NormParams p, const NormLayout l) {
  constexpr bool kHold = NU <= 3;  // g and h of the row stay in registers between its two uses
  extern __shared__ __align__(16) uint8_t smem[];
  float* w = reinterpret_cast<float*>(smem);
  const Team team(l.warps);
  const int c0 = lane_col<VEC, NU>(team), full = full_units<NU>(team, p.C);
  uint8_t* ring = smem + l.params + team.id * l.team_bytes;
  float* red = reinterpret_cast<float*>(ring + l.team_bytes) - 16;  // the last 64 bytes of the team's part
  constexpr int kT = static_cast<int>(sizeof(T));
  const int nb = static_cast<int>(pack_blocks(p.C)), bytes = p.C * kT, xbytes = PACKED ? nb * kPackBlock : bytes;
  const int off_x = row_slot(l.cols * kT), off_s = off_x + row_slot(PACKED ? l.cols : l.cols * kT);
  const uint8_t* const ybase = static_cast<const uint8_t*>(p.dy);
  const uint8_t* const xbase = PACKED ? reinterpret_cast<const uint8_t*>(p.codes) : static_cast<const uint8_t*>(p.x);
  const long long yrow = p.dy_stride * kT, xrow = PACKED ? xbytes : p.x_stride * kT;
  const int step = gridDim.x * l.teams, first = blockIdx.x * l.teams + team.id;
  long long fetched = first;
  int into = 0;
  auto fetch = [&] {
    if (fetched < p.T) {
      uint8_t* dst = ring + into * l.slot;
      fetch_row(ybase + fetched * yrow, bytes, ybase, dst, team.t, team.n);
      fetch_row(xbase + fetched * xrow, xbytes, xbase, dst + off_x, team.t, team.n);
      if constexpr (PACKED) fetch_row(p.scales + fetched * nb, nb, p.scales, dst + off_s, team.t, team.n);
    }
    copies_commit();
    fetched += step;
    into = into + 1 == kPasses ? 0 : into + 1;
  };
  for (int k = 0; k < kPasses; ++k) {
    uint8_t* slot = ring + k * l.slot;
    clear_tail(slot, bytes, off_x, team);
    clear_tail(slot + off_x, xbytes, off_s - off_x, team);
    if constexpr (PACKED) clear_tail(slot + off_s, nb, l.slot - off_s, team);
  }
  team.sync();
  griddep_wait();
  for (int k = 0; k < kPasses - 1; ++k) fetch();
  stage_param<T, VEC>(w, p.w, p.w_f32, 1.f, p.C, l.cols);
  __syncthreads();
  const float inv_c = 1.f / static_cast<float>(p.C);
  uint64_t dw[NU][4], db[NU][4];  // pairs of neighbouring columns
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int e = 0; e < 4; ++e) dw[u][e] = db[u][e] = 0;
  float nmean = first < p.T ? __ldcg(p.mean + first) : 0.f, nrstd = first < p.T ? __ldcg(p.rstd + first) : 0.f;
  int at = 0;
  for (long long row = first; row < p.T; row += step) {
    const float mean = nmean, rstd = nrstd;
    if (row + step < p.T) {
      nmean = __ldcg(p.mean + row + step);
      nrstd = __ldcg(p.rstd + row + step);
    }
    copies_wait<kPasses - 2>();
    team.sync();  // the row is in the ring, and nobody reads the one before it any more
    fetch();
    const uint8_t* slot = ring + at * l.slot;
    const uint8_t* sy = slot + lead(ybase + row * yrow);
    const uint8_t* sx = slot + off_x + (PACKED ? 0 : lead(xbase + row * xrow));
    const uint8_t* ss = slot + off_s + (PACKED ? lead(p.scales + row * nb) : 0);
    const uint64_t nmean2 = both(-mean), rstd2 = both(rstd);
    // unit u: dy, g = dy w and h = (x - mean) rstd, in pairs (dy and g are zero past column C)
    auto values = [&](int u, uint64_t (&d)[4], uint64_t (&g)[4], uint64_t (&h)[4]) {
      float a[8], x[8], ww[8];
      unit_get<T, VEC>(sy, c0, u, a);
      if constexpr (PACKED) unit_get_packed<VEC>(sx, ss, c0, u, x);
      else unit_get<T, VEC>(sx, c0, u, x);
      unit_param<VEC>(w, c0, u, l.cols, ww);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d[e] = f2pack(a[2 * e], a[2 * e + 1]);
        g[e] = mul2(d[e], f2pack(ww[2 * e], ww[2 * e + 1]));
        h[e] = mul2(add2(f2pack(x[2 * e], x[2 * e + 1]), nmean2), rstd2);
      }
    };
    uint64_t s1 = 0, s2 = 0;
    uint64_t keep_g[kHold ? NU : 1][4], keep_h[kHold ? NU : 1][4];
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if constexpr (!kHold) asm volatile("" ::: "memory");  // one unit's loads at a time: the sums take the registers
      uint64_t d[4], g[4], h[4];
      values(u, d, g, h);
      if constexpr (kHold) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          keep_g[u][e] = g[e];
          keep_h[u][e] = h[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        dw[u][e] = fma2(d[e], h[e], dw[u][e]);
        db[u][e] = add2(db[u][e], d[e]);
        s1 = add2(s1, g[e]);
        s2 = fma2(g[e], h[e], s2);
      }
    }
    float s[2], t0, t1;
    f2unpack(s1, t0, t1);
    s[0] = t0 + t1;
    f2unpack(s2, t0, t1);
    s[1] = t0 + t1;
    team.sum(s, red);
    const uint64_t c1 = both(-s[0] * inv_c), c2 = both(-s[1] * inv_c);
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      uint64_t g[4], h[4];
      if constexpr (kHold) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          g[e] = keep_g[u][e];
          h[e] = keep_h[u][e];
        }
      } else {
        asm volatile("" ::: "memory");
        uint64_t d[4];
        values(u, d, g, h);
      }
      float o[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) f2unpack(mul2(fma2(h[e], c2, add2(g[e], c1)), rstd2), o[2 * e], o[2 * e + 1]);
      unit_put<T, VEC>(out, c0, u, full, p.C, o);
    }
    at = at + 1 == kPasses ? 0 : at + 1;
  }
  if (!p.partial) return;
  // the block's teams add their columns' sums: each in its own part of shared memory
  copies_wait<0>();
  __syncthreads();
  float* mine = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int u = 0; u < NU; ++u)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = unit_col<VEC>(c0, u, j / VEC) + j % VEC;
      float a0, a1, b0, b1;
      f2unpack(dw[u][j / 2], a0, a1);
      f2unpack(db[u][j / 2], b0, b1);
      if (c < p.C) {
        mine[c] = j & 1 ? a1 : a0;
        mine[p.C + c] = j & 1 ? b1 : b0;
      }
    }
  __syncthreads();
  float* part = p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.C;
  for (int c = threadIdx.x; c < 2 * p.C; c += blockDim.x) {
    float sum = 0.f;
    for (int q = 0; q < l.teams; ++q) sum += reinterpret_cast<const float*>(smem + l.params + q * l.team_bytes)[c];
    part[c] = sum;
  }
}

// More than 8192 columns: dx by one block per row (the row is read twice), the
// weight gradients by one thread per column over a strip of rows.
template <typename T, bool PACKED>
__device__ __forceinline__ float wide_x(const NormParams& p, long long row, int c) {
  if constexpr (PACKED) {
    const long long nb = pack_blocks(p.C);
    return static_cast<float>(__ldcg(p.codes + row * nb * kPackBlock + c)) * pack_step(__ldcg(p.scales + row * nb + c / kPackBlock));
  } else {
    return elem_f32<T>(static_cast<const T*>(p.x)[row * p.x_stride + c]);
  }
}

template <typename T, bool PACKED>
__global__ void __launch_bounds__(1024) layer_norm_bwd_wide_kernel(const NormParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  __shared__ float red[2][64];
  const float inv_c = 1.f / static_cast<float>(p.C);
  int phase = 0;
  for (long long row = blockIdx.x; row < p.T; row += gridDim.x, phase ^= 1) {
    const float mean = __ldcg(p.mean + row), rstd = __ldcg(p.rstd + row);
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      const float g = elem_f32<T>(dy[c]) * param_at(p.w, p.w_f32, kBf16, c, 1.f);
      s[0] += g;
      s[1] += g * (wide_x<T, PACKED>(p, row, c) - mean) * rstd;
    }
    block_sum<2>(s, red[phase]);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      const float g = elem_f32<T>(dy[c]) * param_at(p.w, p.w_f32, kBf16, c, 1.f);
      out[c] = f32_elem<T>(rstd * (g - c1 - (wide_x<T, PACKED>(p, row, c) - mean) * rstd * c2));
    }
  }
}

template <typename T, bool PACKED>
__global__ void __launch_bounds__(256) layer_norm_bwd_wide_cols_kernel(const NormParams p) {
  griddep_wait();
  griddep_launch_dependents();
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= p.C) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < p.T; row += gridDim.y) {
    const float d = elem_f32<T>(static_cast<const T*>(p.dy)[row * p.dy_stride + c]);
    dw += d * (wide_x<T, PACKED>(p, row, c) - __ldcg(p.mean + row)) * __ldcg(p.rstd + row);
    db += d;
  }
  p.partial[static_cast<size_t>(blockIdx.y) * 2 * p.C + c] = dw;
  p.partial[(static_cast<size_t>(blockIdx.y) * 2 + 1) * p.C + c] = db;
}

// out_a[c] = sum over g < groups of partial[g][a][c], a < arrays: 32 columns and
// 32 row lanes per block, the lanes' sums joined in a fixed order. Behind act_bwd_kernel
// and the wide kernels its blocks start while those still run (programmatic dependent
// launch), behind layer_norm_bwd_kernel as that one ends.
struct FinishParams {
  const float* partial;
  int groups, arrays, C;
  void* out[2];
  int dtype;  // of the outputs
};

__global__ void __launch_bounds__(1024) column_finish_kernel(const FinishParams p) {
  __shared__ float red[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x, a = blockIdx.y;
  griddep_wait();
  griddep_launch_dependents();
  float s = 0.f;
  if (c < p.C) {
    for (int g0 = threadIdx.y; g0 < p.groups; g0 += 32 * 8) {
      float v[8];  // (all in flight together)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int g = g0 + 32 * i;
        v[i] = g < p.groups ? __ldcg(p.partial + (static_cast<size_t>(g) * p.arrays + a) * p.C + c) : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
  }
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  // one warp per column: lane g holds row lane g's sum
  s = red[threadIdx.x][threadIdx.y];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  const int d = blockIdx.x * 32 + threadIdx.y;
  void* out = a ? p.out[1] : p.out[0];
  if (threadIdx.x || d >= p.C || !out) return;
  if (p.dtype == FRATTN_F32) static_cast<float*>(out)[d] = s;
  else if (p.dtype == FRATTN_BF16) static_cast<__nv_bfloat16*>(out)[d] = __float2bfloat16_rn(s);
  else static_cast<__half*>(out)[d] = __float2half_rn(s);
}

// ---------------------------------------------------------------- checkpoints
struct PackParams {
  const void* x;
  long long x_stride;
  int8_t* codes;
  uint8_t* scales;
  void* out;
  long long out_stride;
  int T, C;
};

// One vector of VEC columns per thread and row, 32 / VEC neighbouring threads per
// block of 32 values. Columns past C (the last block of a row) are zeros.
template <typename T, int VEC>
__global__ void __launch_bounds__(256, 8) act_pack_kernel(const PackParams p) {
  constexpr int G = kPackBlock / VEC;  // threads of a block of 32
  constexpr int R = 1;  // (the warps of a full SM keep enough on its way; 4 rows to a thread took half as long again)
  const int nb = static_cast<int>(pack_blocks(p.C));
  const int v = blockIdx.x * blockDim.x + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  const bool in_row = v < nb * G;  // uniform within a block of 32 values
  const bool has = v * VEC < p.C;
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  // (blockDim.x is a multiple of 32, so a warp's lanes share their rows and its shuffles are whole)
  for (long long row0 = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; row0 < p.T; row0 += step * R) {
    Vec<T, VEC> x[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (has && row < p.T) x[r].load(static_cast<const T*>(p.x) + row * p.x_stride + static_cast<size_t>(v) * VEC);
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      float f[VEC];
      x[r].get(f);
      if (!has) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) f[e] = 0.f;
      }
      float m = 0.f;
#pragma unroll
      for (int e = 0; e + 1 < VEC; e += 2) m = max3_abs(m, f[e], f[e + 1]);
      if constexpr (VEC == 1) m = fabsf(f[0]);
      uint32_t amax = abs_bits(m);  // (as integers a NaN is the largest)
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const uint32_t scale = pack_scale(amax);
      if (in_row && row < p.T) {
        int8_t* dst = p.codes + row * nb * kPackBlock + static_cast<size_t>(v) * VEC;
        const float inv = pack_inv(scale);
        if constexpr (VEC == 1) {
          *dst = static_cast<int8_t>(pack_code(f[0], inv, pack_limit(scale)));
        } else if constexpr (VEC == 2) {
          const float lim = pack_limit(scale);
          *reinterpret_cast<uint16_t*>(dst) =
              static_cast<uint16_t>(__byte_perm(pack_code(f[0], inv, lim), pack_code(f[1], inv, lim), 0x0040));
        } else {
          uint32_t codes[VEC / 4];
          pack_codes<VEC>(f, __uint_as_float(amax), scale, codes);
          if constexpr (VEC == 4) *reinterpret_cast<uint32_t*>(dst) = codes[0];
          else *reinterpret_cast<uint2*>(dst) = make_uint2(codes[0], codes[1]);
        }
        if (v % G == 0) p.scales[row * nb + v / G] = static_cast<uint8_t>(scale);
      }
    }
  }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(256) act_unpack_kernel(const PackParams p) {
  constexpr int R = 4;
  const int nb = static_cast<int>(pack_blocks(p.C));
  const int v = blockIdx.x * blockDim.x + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  if (v * VEC >= p.C) return;
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  for (long long row0 = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; row0 < p.T; row0 += step * R) {
    CodeVec<VEC> in[R];
    uint32_t scale[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row < p.T) {
        in[r].load(p.codes + row * nb * kPackBlock + static_cast<size_t>(v) * VEC);
        scale[r] = __ldcg(p.scales + row * nb + v * VEC / kPackBlock);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row >= p.T) break;
      float f[VEC];
      in[r].get(pack_step(scale[r]), f);
      Vec<T, VEC>::put(static_cast<T*>(p.out) + row * p.out_stride + static_cast<size_t>(v) * VEC, f);
    }
  }
}

int sms() {
  const int n = sm_count_for_current_device();
  return n > 0 ? n : 148;
}

constexpr int kMaxCols = 8192;  // widest row held in registers (8 warps of 1024 columns)

constexpr int kSmemPerSm = 227 * 1024;

// Calls f<VEC, NU>() for rows of C columns read in vectors of vec by teams of `warps`.
template <int VEC, typename F>
int with_units(int units, F&& f) {
  switch (units) {
    case 1: return f(std::integral_constant<int, VEC>(), std::integral_constant<int, 1>());
    case 2: return f(std::integral_constant<int, VEC>(), std::integral_constant<int, 2>());
    case 3: return f(std::integral_constant<int, VEC>(), std::integral_constant<int, 3>());
    case 4: return f(std::integral_constant<int, VEC>(), std::integral_constant<int, 4>());
    default: return f(std::integral_constant<int, VEC>(), std::integral_constant<int, 5>());
  }
}
template <typename F>
int with_shape(int vec, int C, int warps, F&& f) {
  const int units = (C + 256 * warps - 1) / (256 * warps);  // of 8 columns to a lane
  if (vec == 8) return with_units<8>(units, f);
  if (vec == 4) return with_units<4>(units, f);
  return with_units<1>(units, f);
}
// Warps to a row of the forward: as few as 40 columns to a lane allow (32 where they are
// single columns, whose addresses take registers too).
int team_warps(int C, int vec) { return vec == 1 ? (C + 1023) / 1024 : (C + 1279) / 1280; }
// Of the backward, whose lanes hold two sums a column besides: a warp for up to 1280
// columns in vectors of 8 (two warps, which have to wait for each other, took 75 us
// where one takes 57 at 32768 x 1280), else 32 columns to a lane. Twelve warps to an SM:
// sixteen leave 128 registers to a thread, and spill (73 us there).
int bwd_team_warps(int C, int vec, bool packed) {
  if (vec == 8 && !packed && C <= 1280) return 1;
  const int w = (C + 1023) / 1024;
  return w < 8 ? w : 8;
}
// With this few rows to an SM latency counts: 8 columns to a lane, up to 8 warps (forward
// of 500 x 6000: 7 us against 12 through the ring).
constexpr int kFewRows = 2, kFewRowsFwd = 4;
int short_team_warps(int C) {
  const int w = (C + 255) / 256;
  return w < 8 ? w : 8;
}

// Teams of a block: as many as fit `threads` and the shared memory of 1 / blocks_per_sm of
// an SM; of these no more than the rows, dealt out evenly, keep busy to the end.
template <typename F>
NormLayout norm_layout(int T, int C, int warps, int threads, int blocks_per_sm, int params, int least_team_bytes,
                       F&& slot_of_cols) {
  NormLayout l;
  l.warps = warps;
  l.cols = 256 * warps * ((C + 256 * warps - 1) / (256 * warps));
  l.params = params * l.cols * 4;
  l.slot = slot_of_cols(l.cols);
  const int most = threads / (32 * warps) < 15 || warps == 1 ? threads / (32 * warps) : 15;  // (named barriers 1 to 15)
  const int room = kSmemPerSm / blocks_per_sm - 1024 - l.params;
  const int ring = kPasses * l.slot > least_team_bytes ? kPasses * l.slot : least_team_bytes;
  l.team_bytes = (ring + 15) / 16 * 16 + 64;  // + the reduction's floats
  const int fit = room / l.team_bytes;
  l.teams = most < fit ? most : fit;
  if (l.teams < 1) l.teams = 1;
  const long long blocks = static_cast<long long>(sms()) * blocks_per_sm;
  const long long rows = (T + blocks * l.teams - 1) / (blocks * l.teams);  // of the busiest team
  l.teams = static_cast<int>((T + blocks * rows - 1) / (blocks * rows));
  return l;
}

// Rings of more than 48 KB are allowed once per kernel and device.
template <typename K>
bool allow_ring(K kern, unsigned long long& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bit = 1ull << (dev & 63);
  if (done & bit) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemPerSm) != cudaSuccess) return false;
  done |= bit;
  return true;
}

int norm_blocks(int T, const NormLayout& l, int blocks_per_sm) {
  const long long want = (static_cast<long long>(T) + l.teams - 1) / l.teams;
  const long long cap = static_cast<long long>(sms()) * blocks_per_sm;
  return static_cast<int>(want < cap ? want : cap);
}

template <typename T>
int norm_fwd(NormParams p, cudaStream_t st) {
  if (p.C > kMaxCols) {
    const int n = p.T < 2 * sms() ? p.T : 2 * sms();
    return launch_overlapped(layer_norm_fwd_wide_kernel<T>, dim3(n), dim3(1024), 0, st, 1, p);
  }
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride).row(p.out, p.out_stride);
  if (rv.v == 2) rv.v = 1;
  if (p.T <= kFewRowsFwd * sms()) {
    p.w_vec = aligned_to(p.w, 16) && aligned_to(p.b, 16);
    const int warps = short_team_warps(p.C);
    return with_shape(rv.v, p.C, warps, [&](auto vec, auto nu) {
      return launch_overlapped(layer_norm_fwd_few_kernel<T, decltype(vec)::value, decltype(nu)::value>, dim3(p.T),
                               dim3(32 * warps), 0, st, 1, p);
    });
  }
  const int warps = team_warps(p.C, rv.v);
  // Blocks of 256 threads to an SM: what the registers allow, fewer where even one team's rows
  // and the parameters take more than that share of the shared memory (16-bit rows from
  // 5121 columns, fp32 from 4097). The rows are dealt out over the blocks that run at once:
  // dealt out over three to an SM where two fit, 9216 x 5376 bf16 took 90 us, so 67.
  int blocks = (p.C + 256 * warps - 1) / (256 * warps) > 3 ? 3 : 4;
  auto layout = [&] {
    return norm_layout(p.T, p.C, warps, 256, blocks, 2, 0,
                       [](int cols) { return row_slot(cols * static_cast<int>(sizeof(T))); });
  };
  NormLayout l = layout();
  while (blocks > 1 && l.params + l.teams * l.team_bytes > kSmemPerSm / blocks - 1024) {
    --blocks;
    l = layout();
  }
  return with_shape(rv.v, p.C, warps, [&](auto vec, auto nu) {
    auto kern = layer_norm_fwd_kernel<T, decltype(vec)::value, decltype(nu)::value>;
    static unsigned long long ring_ok = 0;
    if (!allow_ring(kern, ring_ok)) return static_cast<int>(FRATTN_E_CUDA);
    return launch_overlapped(kern, dim3(norm_blocks(p.T, l, blocks)), dim3(32 * l.warps * l.teams),
                             l.params + l.teams * l.team_bytes, st, 1, p, l);
  });
}

template <typename T, bool PACKED>
int norm_bwd(const NormParams& p, int* groups, cudaStream_t st) {
  if (p.C > kMaxCols) {
    const int n = p.T < 2 * sms() ? p.T : 2 * sms();
    const int rc = launch_overlapped(layer_norm_bwd_wide_kernel<T, PACKED>, dim3(n), dim3(1024), 0, st, 1, p);
    if (rc || !p.partial) return rc;
    *groups = p.T < sms() ? p.T : sms();
    return launch_overlapped(layer_norm_bwd_wide_cols_kernel<T, PACKED>, dim3((p.C + 255) / 256, *groups), dim3(256), 0, st,
                             1, p);
  }
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride).row(p.dy, p.dy_stride).row(p.out, p.out_stride);
  if (rv.v == 2) rv.v = 1;
  const int warps = p.T <= kFewRows * sms() ? short_team_warps(p.C) : bwd_team_warps(p.C, rv.v, PACKED);
  const int gradients = 2 * p.C * 4;  // a team's, in the end
  const NormLayout l = norm_layout(p.T, p.C, warps, 384, 1, 1, gradients, [](int cols) {
    const int row = row_slot(cols * static_cast<int>(sizeof(T)));
    return row + (PACKED ? row_slot(cols) + row_slot(cols / kPackBlock) : row);
  });
  return with_shape(rv.v, p.C, l.warps, [&](auto vec, auto nu) {
    auto kern = layer_norm_bwd_kernel<T, decltype(vec)::value, decltype(nu)::value, PACKED>;
    static unsigned long long ring_ok = 0;
    if (!allow_ring(kern, ring_ok)) return static_cast<int>(FRATTN_E_CUDA);
    *groups = norm_blocks(p.T, l, 1);
    return launch_overlapped(kern, dim3(*groups), dim3(32 * l.warps * l.teams), l.params + l.teams * l.team_bytes, st, 1,
                             p, l);
  });
}

// Launch shape of the checkpoint kernels for nv vectors per row.
void pack_shape(int nv, int T, dim3* grid, dim3* block) {
  int bx;
  if (nv >= 32) {
    const int tiles = (nv + 255) / 256;
    bx = ((nv + tiles - 1) / tiles + 31) / 32 * 32;
  } else {
    bx = 32;
  }
  const int by = 256 / bx > 0 ? 256 / bx : 1;
  *block = dim3(bx, by);
  const int gx = (nv + bx - 1) / bx;
  const long long want = (static_cast<long long>(T) + 4 * by - 1) / (4 * by);
  const long long cap = (static_cast<long long>(sms()) * 32 + gx - 1) / gx;
  long long gy = want < cap ? want : cap;
  if (gy > 65535) gy = 65535;
  *grid = dim3(gx, static_cast<unsigned>(gy));
}

template <typename T>
int pack(const PackParams& p, cudaStream_t st) {
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride);
  dim3 grid, block;
  const int nb = static_cast<int>(pack_blocks(p.C));
  pack_shape(nb * (kPackBlock / rv.v), p.T, &grid, &block);
  if (rv.v == 8) return launch_overlapped(act_pack_kernel<T, 8>, grid, block, 0, st, 1, p);
  if (rv.v == 4) return launch_overlapped(act_pack_kernel<T, 4>, grid, block, 0, st, 1, p);
  if (rv.v == 2) return launch_overlapped(act_pack_kernel<T, 2>, grid, block, 0, st, 1, p);
  return launch_overlapped(act_pack_kernel<T, 1>, grid, block, 0, st, 1, p);
}

template <typename T>
int unpack(const PackParams& p, cudaStream_t st) {
  RowVec rv(p.C, sizeof(T));
  rv.row(p.out, p.out_stride);
  dim3 grid, block;
  pack_shape((p.C + rv.v - 1) / rv.v, p.T, &grid, &block);
  if (rv.v == 8) return launch_overlapped(act_unpack_kernel<T, 8>, grid, block, 0, st, 1, p);
  if (rv.v == 4) return launch_overlapped(act_unpack_kernel<T, 4>, grid, block, 0, st, 1, p);
  if (rv.v == 2) return launch_overlapped(act_unpack_kernel<T, 2>, grid, block, 0, st, 1, p);
  return launch_overlapped(act_unpack_kernel<T, 1>, grid, block, 0, st, 1, p);
}

bool known_dtype(int d) { return d == FRATTN_F32 || d == FRATTN_F16 || d == FRATTN_BF16; }

}  // namespace

// Sums of partial rows (also for the linear layer's bias gradient).
int column_finish(const float* partial, int groups, int arrays, int C, void* out0, void* out1, int dtype,
                  cudaStream_t st) {
  FinishParams f;
  f.partial = partial;
  f.groups = groups;
  f.arrays = arrays;
  f.C = C;
  f.out[0] = out0;
  f.out[1] = out1;
  f.dtype = dtype;
  return launch_overlapped(column_finish_kernel, dim3((C + 31) / 32, arrays), dim3(32, 32), 0, st, 1, f);
}

// Checkpoint of a matrix back to 16-bit values (the linear layer's backward pass).
int act_unpack(const int8_t* codes, const uint8_t* scales, int T, int C, int dtype, void* out, long long out_stride,
               cudaStream_t st) {
  PackParams p;
  memset(&p, 0, sizeof(p));
  p.codes = const_cast<int8_t*>(codes);
  p.scales = const_cast<uint8_t*>(scales);
  p.out = out;
  p.out_stride = out_stride;
  p.T = T;
  p.C = C;
  if (dtype == FRATTN_F32) return unpack<float>(p, st);
  if (dtype == FRATTN_BF16) return unpack<__nv_bfloat16>(p, st);
  return unpack<__half>(p, st);
}

}  // namespace frattn

using namespace frattn;

extern "C" {

int frattn_layer_norm(const void* x, long long x_stride, const void* weight, const void* bias, int param_dtype, int T,
                      int C, float eps, int dtype, void* out, long long out_stride, float* mean, float* rstd,
                      void* stream) {
  if (T < 0 || C <= 0 || x_stride < 0 || out_stride < C || !(eps >= 0.f)) return FRATTN_E_SHAPE;
  if (!known_dtype(dtype) || (param_dtype != dtype && param_dtype != FRATTN_F32)) return FRATTN_E_DTYPE;
  if (T == 0) return 0;
  if (!x || !out) return FRATTN_E_NULL;
  const int es = dtype == FRATTN_F32 ? 4 : 2, ps = param_dtype == FRATTN_F32 ? 4 : 2;
  if (!aligned_to(x, es) || !aligned_to(out, es) || !aligned_to(weight, ps) || !aligned_to(bias, ps) ||
      !aligned_to(mean, 4) || !aligned_to(rstd, 4))
    return FRATTN_E_ALIGN;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = x;
  p.x_stride = x_stride;
  p.w = weight;
  p.b = bias;
  p.w_f32 = param_dtype == FRATTN_F32;
  p.out = out;
  p.out_stride = out_stride;
  p.mean = mean;
  p.rstd = rstd;
  p.T = T;
  p.C = C;
  p.eps = eps;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FRATTN_F32) return norm_fwd<float>(p, st);
  if (dtype == FRATTN_BF16) return norm_fwd<__nv_bfloat16>(p, st);
  return norm_fwd<__half>(p, st);
}

int frattn_workspace_bytes_layer_norm_bwd(int T, int C, size_t* bytes) {
  if (!bytes) return FRATTN_E_NULL;
  if (T < 0 || C <= 0) return FRATTN_E_SHAPE;
  // one partial row of the two weight gradients per block
  const long long blocks = sms();
  *bytes = static_cast<size_t>(T < blocks ? (T > 0 ? T : 1) : blocks) * 2 * C * sizeof(float);
  return 0;
}

int frattn_layer_norm_bwd(const void* dout, long long dout_stride, const void* x, long long x_stride,
                          const int8_t* codes, const uint8_t* scales, const void* weight, int param_dtype,
                          const float* mean, const float* rstd, int T, int C, int dtype, void* dx,
                          long long dx_stride, void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                          void* stream) {
  if (T < 0 || C <= 0 || dout_stride < 0 || x_stride < 0 || dx_stride < C) return FRATTN_E_SHAPE;
  if (!known_dtype(dtype) || (param_dtype != dtype && param_dtype != FRATTN_F32)) return FRATTN_E_DTYPE;
  const bool want = dweight || dbias;
  if (T > 0 && (!dout || !dx || !mean || !rstd || (x ? codes || scales : !codes || !scales))) return FRATTN_E_NULL;
  if (want && !workspace) return FRATTN_E_NULL;
  const int es = dtype == FRATTN_F32 ? 4 : 2, ps = param_dtype == FRATTN_F32 ? 4 : 2;
  if (!aligned_to(x, es) || !aligned_to(dout, es) || !aligned_to(dx, es) || !aligned_to(codes, 16) ||
      !aligned_to(weight, ps) || !aligned_to(dweight, ps) || !aligned_to(dbias, ps) || !aligned_to(mean, 4) ||
      !aligned_to(rstd, 4) || !aligned_to(workspace, 16))
    return FRATTN_E_ALIGN;
  size_t need = 0;
  frattn_workspace_bytes_layer_norm_bwd(T, C, &need);
  if (want && workspace_bytes < need) return FRATTN_E_WORKSPACE;
  NormParams p;
  memset(&p, 0, sizeof(p));
  p.x = x;
  p.x_stride = x_stride;
  p.codes = codes;
  p.scales = scales;
  p.w = weight;
  p.w_f32 = param_dtype == FRATTN_F32;
  p.dy = dout;
  p.dy_stride = dout_stride;
  p.out = dx;
  p.out_stride = dx_stride;
  p.mean = const_cast<float*>(mean);
  p.rstd = const_cast<float*>(rstd);
  p.partial = want ? static_cast<float*>(workspace) : nullptr;
  p.T = T;
  p.C = C;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  int groups = 0, rc = 0;
  if (T > 0) {
    if (dtype == FRATTN_F32) rc = x ? norm_bwd<float, false>(p, &groups, st) : norm_bwd<float, true>(p, &groups, st);
    else if (dtype == FRATTN_BF16)
      rc = x ? norm_bwd<__nv_bfloat16, false>(p, &groups, st) : norm_bwd<__nv_bfloat16, true>(p, &groups, st);
    else rc = x ? norm_bwd<__half, false>(p, &groups, st) : norm_bwd<__half, true>(p, &groups, st);
  }
  if (rc || !want) return rc;
  return column_finish(p.partial, groups, 2, C, dweight, dbias, param_dtype, st);
}

int frattn_act_pack(const void* x, long long x_stride, int T, int C, int dtype, int8_t* codes, uint8_t* scales,
                    void* stream) {
  if (T < 0 || C <= 0 || C > (1 << 30) || x_stride < 0) return FRATTN_E_SHAPE;
  if (!known_dtype(dtype)) return FRATTN_E_DTYPE;
  if (T == 0) return 0;
  if (!x || !codes || !scales) return FRATTN_E_NULL;
  if (!aligned_to(x, dtype == FRATTN_F32 ? 4 : 2) || !aligned_to(codes, 16)) return FRATTN_E_ALIGN;
  PackParams p;
  memset(&p, 0, sizeof(p));
  p.x = x;
  p.x_stride = x_stride;
  p.codes = codes;
  p.scales = scales;
  p.T = T;
  p.C = C;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == FRATTN_F32) return pack<float>(p, st);
  if (dtype == FRATTN_BF16) return pack<__nv_bfloat16>(p, st);
  return pack<__half>(p, st);
}

int frattn_act_unpack(const int8_t* codes, const uint8_t* scales, int T, int C, int dtype, void* out,
                      long long out_stride, void* stream) {
  if (T < 0 || C <= 0 || C > (1 << 30) || out_stride < C) return FRATTN_E_SHAPE;
  if (!known_dtype(dtype)) return FRATTN_E_DTYPE;
  if (T == 0) return 0;
  if (!codes || !scales || !out) return FRATTN_E_NULL;
  if (!aligned_to(out, dtype == FRATTN_F32 ? 4 : 2) || !aligned_to(codes, 16)) return FRATTN_E_ALIGN;
  return act_unpack(codes, scales, T, C, dtype, out, out_stride, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
