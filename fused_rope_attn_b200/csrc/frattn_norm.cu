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
// Both are bound by the bytes of the rows. One block holds R whole rows in
// registers (one vector of up to 8 columns per thread for rows of up to 8192
// columns), so every row is read once; R = 4 rows share each block-wide
// reduction's barrier and keep four rows' loads in flight. The weight
// gradients stay in the registers of the thread that owns the column over all
// rows of a block; each block writes one partial row, and column_finish adds
// the partial rows in a fixed order (no atomics: the same bits every run).
#include "frattn_block.cuh"

namespace frattn {

struct NormParams {
  const void* x;        // [T, C] rows of x_stride elements (null: codes / scales)
  long long x_stride;
  const int8_t* codes;  // [T, 32 nb]
  const uint8_t* scales;  // [T, nb]
  const void* w;        // [C] or null (ones)
  const void* b;        // [C] or null (zeros), forward only
  int w_f32;            // w, b, dw, db are fp32 (else the element type)
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

// Sums over the block's threads of R values; every thread gets them. `red` holds
// R x 32 floats and must not be reused before the next barrier but one.
template <int R>
__device__ __forceinline__ void block_sum(float (&s)[R], float* red) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return;
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
#pragma unroll
    for (int r = 0; r < R; ++r) red[r * 32 + warp] = s[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float t = 0.f;
    for (int w = 0; w < nw; ++w) t += red[r * 32 + w];
    s[r] = t;
  }
}

// Parameter vector (weight or bias) of columns [c, c + VEC) in 32 bits.
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, int f32, int c, float fill, float (&v)[VEC]) {
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    if (!p) v[e] = fill;
    else v[e] = f32 ? __ldg(static_cast<const float*>(p) + c + e) : elem_f32<T>(static_cast<const T*>(p)[c + e]);
  }
}

template <typename T, int VEC, int NV, int R>
__global__ void __launch_bounds__(R == 1 ? 1024 : 512) layer_norm_fwd_kernel(const NormParams p) {
  __shared__ float red[2][R * 32];
  const int nvec = p.C / VEC;
  float w[NV][VEC], b[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) {
      load_param<T, VEC>(p.w, p.w_f32, v * VEC, 1.f, w[i]);
      load_param<T, VEC>(p.b, p.w_f32, v * VEC, 0.f, b[i]);
    }
  }
  const float inv_c = 1.f / static_cast<float>(p.C);
  for (long long row0 = static_cast<long long>(blockIdx.x) * R; row0 < p.T; row0 += static_cast<long long>(gridDim.x) * R) {
    Vec<T, VEC> x[R][NV];
    float s[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const T* row = static_cast<const T*>(p.x) + (row0 + r) * p.x_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < nvec && row0 + r < p.T) x[r][i].load(row + static_cast<size_t>(v) * VEC);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (static_cast<int>(threadIdx.x + i * blockDim.x) < nvec && row0 + r < p.T) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[r] += x[r][i].get(e);
        }
    }
    block_sum<R>(s, red[0]);
    float mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = s[r] * inv_c;
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (static_cast<int>(threadIdx.x + i * blockDim.x) < nvec && row0 + r < p.T) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float d = x[r][i].get(e) - mean[r];
            s[r] += d * d;
          }
        }
    }
    block_sum<R>(s, red[1]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r;
      if (row >= p.T) break;
      const float rstd = rsqrtf(s[r] * inv_c + p.eps);
      if (threadIdx.x == 0) {
        if (p.mean) p.mean[row] = mean[r];
        if (p.rstd) p.rstd[row] = rstd;
      }
      T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < nvec) {
          Vec<T, VEC> y;
#pragma unroll
          for (int e = 0; e < VEC; ++e) y.set(e, (x[r][i].get(e) - mean[r]) * rstd * w[i][e] + b[i][e]);
          y.store(out + static_cast<size_t>(v) * VEC);
        }
      }
    }
  }
}

// Rows of more than 8192 columns: one block per row, the row is read three times
// (from L2 after the first).
template <typename T>
__global__ void __launch_bounds__(1024) layer_norm_fwd_wide_kernel(const NormParams p) {
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
      float w[1], b[1];
      load_param<T, 1>(p.w, p.w_f32, c, 1.f, w);
      load_param<T, 1>(p.b, p.w_f32, c, 0.f, b);
      out[c] = f32_elem<T>((elem_f32<T>(x[c]) - mean) * rstd * w[0] + b[0]);
    }
  }
}

// VEC values of an input row: 16/32-bit elements or checkpoint codes.
template <typename T, int VEC, bool PACKED>
struct NormIn {
  Vec<T, VEC> v;
  __device__ __forceinline__ void load(const NormParams& p, long long row, int vec) {
    v.load(static_cast<const T*>(p.x) + row * p.x_stride + static_cast<size_t>(vec) * VEC);
  }
  __device__ __forceinline__ float get(int e) const { return v.get(e); }
};
template <typename T, int VEC>
struct NormIn<T, VEC, true> {
  union {
    typename RawVec<VEC == 1 ? 2 : VEC>::type raw;
    int8_t c[VEC == 1 ? 2 : VEC];
  };
  uint32_t scale;
  __device__ __forceinline__ NormIn() {}
  __device__ __forceinline__ void load(const NormParams& p, long long row, int vec) {
    const long long nb = pack_blocks(p.C);
    const int8_t* src = p.codes + row * nb * kPackBlock + static_cast<size_t>(vec) * VEC;
    if constexpr (VEC == 1) c[0] = __ldg(src);
    else raw = __ldg(reinterpret_cast<const typename RawVec<VEC>::type*>(src));
    scale = __ldg(p.scales + row * nb + vec * VEC / kPackBlock);
  }
  __device__ __forceinline__ float get(int e) const { return static_cast<float>(c[e]) * pack_step(scale); }
};

template <typename T, int VEC, int NV, int R, bool PACKED>
__global__ void __launch_bounds__(R == 1 ? 1024 : 512) layer_norm_bwd_kernel(const NormParams p) {
  __shared__ float red[2][2 * R * 32];
  const int nvec = p.C / VEC;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nvec) load_param<T, VEC>(p.w, p.w_f32, v * VEC, 1.f, w[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const float inv_c = 1.f / static_cast<float>(p.C);
  int phase = 0;
  for (long long row0 = static_cast<long long>(blockIdx.x) * R; row0 < p.T;
       row0 += static_cast<long long>(gridDim.x) * R, phase ^= 1) {
    NormIn<T, VEC, PACKED> x[R][NV];
    Vec<T, VEC> dy[R][NV];
    float mean[R], rstd[R], s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r;
      const bool in = row < p.T;
      mean[r] = in ? __ldg(p.mean + row) : 0.f;
      rstd[r] = in ? __ldg(p.rstd + row) : 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < nvec && in) {
          x[r][i].load(p, row, v);
          dy[r][i].load(static_cast<const T*>(p.dy) + row * p.dy_stride + static_cast<size_t>(v) * VEC);
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (static_cast<int>(threadIdx.x + i * blockDim.x) < nvec && row0 + r < p.T) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float d = dy[r][i].get(e), h = (x[r][i].get(e) - mean[r]) * rstd[r], g = d * w[i][e];
            s[2 * r] += g;
            s[2 * r + 1] += g * h;
            dw[i][e] += d * h;
            db[i][e] += d;
          }
        }
    }
    block_sum<2 * R>(s, red[phase]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r;
      if (row >= p.T) break;
      const float c1 = s[2 * r] * inv_c, c2 = s[2 * r + 1] * inv_c;
      T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
        if (v < nvec) {
          Vec<T, VEC> o;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float h = (x[r][i].get(e) - mean[r]) * rstd[r];
            o.set(e, rstd[r] * (dy[r][i].get(e) * w[i][e] - c1 - h * c2));
          }
          o.store(out + static_cast<size_t>(v) * VEC);
        }
      }
    }
  }
  if (p.partial) {
    float* mine = p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nvec) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          mine[static_cast<size_t>(v) * VEC + e] = dw[i][e];
          mine[p.C + static_cast<size_t>(v) * VEC + e] = db[i][e];
        }
      }
    }
  }
}

// More than 8192 columns: dx by one block per row (the row is read twice), the
// weight gradients by one thread per column over a strip of rows.
template <typename T, bool PACKED>
__global__ void __launch_bounds__(1024) layer_norm_bwd_wide_kernel(const NormParams p) {
  __shared__ float red[2][64];
  const float inv_c = 1.f / static_cast<float>(p.C);
  int phase = 0;
  for (long long row = blockIdx.x; row < p.T; row += gridDim.x, phase ^= 1) {
    const float mean = __ldg(p.mean + row), rstd = __ldg(p.rstd + row);
    const T* dy = static_cast<const T*>(p.dy) + row * p.dy_stride;
    T* out = static_cast<T*>(p.out) + row * p.out_stride;
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      float w[1];
      load_param<T, 1>(p.w, p.w_f32, c, 1.f, w);
      NormIn<T, 1, PACKED> x;
      x.load(p, row, c);
      const float g = elem_f32<T>(dy[c]) * w[0];
      s[0] += g;
      s[1] += g * (x.get(0) - mean) * rstd;
    }
    block_sum<2>(s, red[phase]);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      float w[1];
      load_param<T, 1>(p.w, p.w_f32, c, 1.f, w);
      NormIn<T, 1, PACKED> x;
      x.load(p, row, c);
      out[c] = f32_elem<T>(rstd * (elem_f32<T>(dy[c]) * w[0] - c1 - (x.get(0) - mean) * rstd * c2));
    }
  }
}

template <typename T, bool PACKED>
__global__ void __launch_bounds__(256) layer_norm_bwd_wide_cols_kernel(const NormParams p) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= p.C) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < p.T; row += gridDim.y) {
    NormIn<T, 1, PACKED> x;
    x.load(p, row, c);
    const float d = elem_f32<T>(static_cast<const T*>(p.dy)[row * p.dy_stride + c]);
    dw += d * (x.get(0) - __ldg(p.mean + row)) * __ldg(p.rstd + row);
    db += d;
  }
  p.partial[static_cast<size_t>(blockIdx.y) * 2 * p.C + c] = dw;
  p.partial[(static_cast<size_t>(blockIdx.y) * 2 + 1) * p.C + c] = db;
}

// out_a[c] = sum over g < groups of partial[g][a][c], a < arrays: 32 columns and
// 16 row lanes per block, the lanes' sums joined in a fixed order.
struct FinishParams {
  const float* partial;
  int groups, arrays, C;
  void* out[2];
  int dtype;  // of the outputs
};

__global__ void __launch_bounds__(512) column_finish_kernel(const FinishParams p) {
  __shared__ float red[16][33];
  const int c = blockIdx.x * 32 + threadIdx.x, a = blockIdx.y;
  float s = 0.f;
  if (c < p.C)
#pragma unroll 4
    for (int g = threadIdx.y; g < p.groups; g += 16)
      s += __ldg(p.partial + (static_cast<size_t>(g) * p.arrays + a) * p.C + c);
  red[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y || c >= p.C || !p.out[a]) return;
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) t += red[i][threadIdx.x];
  if (p.dtype == FRATTN_F32) static_cast<float*>(p.out[a])[c] = t;
  else if (p.dtype == FRATTN_BF16) static_cast<__nv_bfloat16*>(p.out[a])[c] = __float2bfloat16_rn(t);
  else static_cast<__half*>(p.out[a])[c] = __float2half_rn(t);
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
__global__ void __launch_bounds__(256) act_pack_kernel(const PackParams p) {
  constexpr int G = kPackBlock / VEC;  // threads of a block of 32
  constexpr int R = 4;
  const int nb = static_cast<int>(pack_blocks(p.C));
  const int v = blockIdx.x * blockDim.x + threadIdx.x;
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
      uint32_t m = 0;
      if (has && row < p.T) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) m = max(m, abs_bits(x[r].get(e)));
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint32_t scale = pack_scale(m);
      const float inv = pack_inv(scale), lim = pack_limit(scale);
      union {
        typename RawVec<VEC == 1 ? 2 : VEC>::type raw;
        int8_t c[VEC == 1 ? 2 : VEC];
      } o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.c[e] = has && row < p.T ? static_cast<int8_t>(pack_code(x[r].get(e), inv, lim)) : 0;
      if (in_row && row < p.T) {
        int8_t* dst = p.codes + row * nb * kPackBlock + static_cast<size_t>(v) * VEC;
        if constexpr (VEC == 1) *dst = o.c[0];
        else *reinterpret_cast<typename RawVec<VEC>::type*>(dst) = o.raw;
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
  if (v * VEC >= p.C) return;
  const long long step = static_cast<long long>(gridDim.y) * blockDim.y;
  for (long long row0 = static_cast<long long>(blockIdx.y) * blockDim.y + threadIdx.y; row0 < p.T; row0 += step * R) {
    union {
      typename RawVec<VEC == 1 ? 2 : VEC>::type raw;
      int8_t c[VEC == 1 ? 2 : VEC];
    } in[R];
    uint32_t scale[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row < p.T) {
        const int8_t* src = p.codes + row * nb * kPackBlock + static_cast<size_t>(v) * VEC;
        if constexpr (VEC == 1) in[r].c[0] = __ldg(src);
        else in[r].raw = __ldg(reinterpret_cast<const typename RawVec<VEC>::type*>(src));
        scale[r] = __ldg(p.scales + row * nb + v * VEC / kPackBlock);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row >= p.T) break;
      const float st = pack_step(scale[r]);
      Vec<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o.set(e, static_cast<float>(in[r].c[e]) * st);
      o.store(static_cast<T*>(p.out) + row * p.out_stride + static_cast<size_t>(v) * VEC);
    }
  }
}

int sms() {
  const int n = sm_count_for_current_device();
  return n > 0 ? n : 148;
}

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : FRATTN_E_CUDA; }

constexpr int kMaxCols = 8192;  // widest row held in registers (1024 threads x 8 columns)

// Threads for nvec vectors, NV to a thread.
int threads_for(int nvec, int nv) { return ((nvec + nv - 1) / nv + 31) / 32 * 32; }

// Vectors to a thread: as few as 1024 threads allow, and at least enough that a
// block of scalar columns stays under 512 threads where it can.
template <typename F>
int with_shape(int vec, int C, F&& f) {
  const int nvec = C / vec;
  if (vec == 8) return f(std::integral_constant<int, 8>(), std::integral_constant<int, 1>(), threads_for(nvec, 1));
  if (vec == 4) return f(std::integral_constant<int, 4>(), std::integral_constant<int, 2>(), threads_for(nvec, 2));
  if (C <= 2048) return f(std::integral_constant<int, 1>(), std::integral_constant<int, 4>(), threads_for(nvec, 4));
  return f(std::integral_constant<int, 1>(), std::integral_constant<int, 8>(), threads_for(nvec, 8));
}

// Rows per block pass: 4 when that still gives every SM a block and the block is
// no larger than 512 threads, else 1 (few rows: latency; long rows: registers).
bool four_rows(int T, int threads) { return threads <= 512 && T >= 4 * sms(); }

int fwd_blocks(int T, int rows, int threads) {
  const long long want = (static_cast<long long>(T) + rows - 1) / rows;
  const long long cap = static_cast<long long>(sms()) * (1536 / threads > 0 ? 1536 / threads : 1);
  return static_cast<int>(want < cap ? want : cap);
}

// Blocks of the backward pass (each writes one partial row of the weight
// gradients). Also the size of the workspace, so a function of T and C alone.
int bwd_blocks(int T, int rows, int threads) {
  const long long want = (static_cast<long long>(T) + rows - 1) / rows;
  const long long cap = static_cast<long long>(sms()) * (768 / threads > 0 ? 768 / threads : 1);
  return static_cast<int>(want < cap ? want : cap);
}
constexpr int kMaxBlocksPerSm = 24;  // 768 / 32

template <typename T>
int norm_fwd(const NormParams& p, cudaStream_t st) {
  if (p.C > kMaxCols) {
    const int n = fwd_blocks(p.T, 1, 1024);
    layer_norm_fwd_wide_kernel<T><<<n, 1024, 0, st>>>(p);
    return launched();
  }
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride).row(p.out, p.out_stride);
  return with_shape(rv.v, p.C, [&](auto vec, auto nv, int threads) {
    constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
    if (four_rows(p.T, threads))
      layer_norm_fwd_kernel<T, V, N, 4><<<fwd_blocks(p.T, 4, threads), threads, 0, st>>>(p);
    else
      layer_norm_fwd_kernel<T, V, N, 1><<<fwd_blocks(p.T, 1, threads), threads, 0, st>>>(p);
    return launched();
  });
}

template <typename T, bool PACKED>
int norm_bwd(NormParams p, int* groups, cudaStream_t st) {
  if (p.C > kMaxCols) {
    const int n = fwd_blocks(p.T, 1, 1024);
    layer_norm_bwd_wide_kernel<T, PACKED><<<n, 1024, 0, st>>>(p);
    if (p.partial) {
      *groups = p.T < sms() ? p.T : sms();
      layer_norm_bwd_wide_cols_kernel<T, PACKED><<<dim3((p.C + 255) / 256, *groups), 256, 0, st>>>(p);
    }
    return launched();
  }
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride).row(p.dy, p.dy_stride).row(p.out, p.out_stride);
  return with_shape(rv.v, p.C, [&](auto vec, auto nv, int threads) {
    constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
    if (four_rows(p.T, threads)) {
      *groups = bwd_blocks(p.T, 4, threads);
      layer_norm_bwd_kernel<T, V, N, 4, PACKED><<<*groups, threads, 0, st>>>(p);
    } else {
      *groups = bwd_blocks(p.T, 1, threads);
      layer_norm_bwd_kernel<T, V, N, 1, PACKED><<<*groups, threads, 0, st>>>(p);
    }
    return launched();
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
  if (rv.v == 8) act_pack_kernel<T, 8><<<grid, block, 0, st>>>(p);
  else if (rv.v == 4) act_pack_kernel<T, 4><<<grid, block, 0, st>>>(p);
  else act_pack_kernel<T, 1><<<grid, block, 0, st>>>(p);
  return launched();
}

template <typename T>
int unpack(const PackParams& p, cudaStream_t st) {
  RowVec rv(p.C, sizeof(T));
  rv.row(p.out, p.out_stride);
  dim3 grid, block;
  pack_shape((p.C + rv.v - 1) / rv.v, p.T, &grid, &block);
  if (rv.v == 8) act_unpack_kernel<T, 8><<<grid, block, 0, st>>>(p);
  else if (rv.v == 4) act_unpack_kernel<T, 4><<<grid, block, 0, st>>>(p);
  else act_unpack_kernel<T, 1><<<grid, block, 0, st>>>(p);
  return launched();
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
  column_finish_kernel<<<dim3((C + 31) / 32, arrays), dim3(32, 16), 0, st>>>(f);
  return launched();
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
  const long long blocks = static_cast<long long>(sms()) * (C <= 1024 ? kMaxBlocksPerSm : 8);
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
