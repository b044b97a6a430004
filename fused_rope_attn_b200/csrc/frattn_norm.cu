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
// Both are bound by the bytes of the rows. A block holds R whole rows in registers
// (one vector of up to 8 columns per thread for rows of up to 8192 columns), so every
// row is read once; the next R rows' loads are issued before the current ones are
// worked on, and R rows share each block-wide reduction's barrier. The weight
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
  int w_vec;            // w and b are 16-byte aligned
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

// Sums over the block's threads of R values (a power of two); every thread gets them.
// Within a warp the lanes split the values among them as they halve: R - 1 + 5 - log2 R
// shuffles instead of 5 R. `red` holds 32 R floats and must not be reused before the
// next barrier but one.
template <int R>
__device__ __forceinline__ void block_sum(float (&s)[R], float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  float t[R];
#pragma unroll
  for (int r = 0; r < R; ++r) t[r] = s[r];
  int o = 16;
#pragma unroll
  for (int n = R; n > 1; n >>= 1, o >>= 1) {
    const bool up = lane & o;  // this lane keeps the upper half of the values
#pragma unroll
    for (int r = 0; r < n / 2; ++r) {
      const float give = up ? t[r] : t[r + n / 2], keep = up ? t[r + n / 2] : t[r];
      t[r] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (int q = 16 / R; q > 0; q >>= 1) t[0] += __shfl_xor_sync(0xffffffffu, t[0], q);
  // value r now lies in the lanes whose bits 4 .. 5 - log2 R spell r (highest bit first)
  if (nw == 1) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] = __shfl_sync(0xffffffffu, t[0], r * (32 / R));
    return;
  }
  if (lane % (32 / R) == 0) red[warp * R + lane / (32 / R)] = t[0];
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) s[r] = 0.f;
  for (int w = 0; w < nw; ++w) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r] += red[w * R + r];
  }
}

// Parameter vector (weight or bias) of columns [c, c + VEC) in 32 bits.
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* p, int f32, int vec, int c, float fill, float (&v)[VEC]) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = fill;
  } else if (vec) {
    if (f32) {
      Vec<float, VEC> x;
      x.load(static_cast<const float*>(p) + c);
      x.get(v);
    } else {
      Vec<T, VEC> x;
      x.load(static_cast<const T*>(p) + c);
      x.get(v);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      v[e] = f32 ? __ldg(static_cast<const float*>(p) + c + e) : elem_f32<T>(static_cast<const T*>(p)[c + e]);
  }
}

template <typename T, int VEC, int NV, int R>
__global__ void __launch_bounds__(R == 1 ? 1024 : R == 2 ? 512 : 256) layer_norm_fwd_kernel(const NormParams p) {
  __shared__ __align__(16) float red[2][R * 32];
  const int nvec = p.C / VEC;
  float w[NV][VEC], b[NV][VEC];
  bool has[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    has[i] = v < nvec;
    if (has[i]) {
      load_param<T, VEC>(p.w, p.w_f32, p.w_vec, v * VEC, 1.f, w[i]);
      load_param<T, VEC>(p.b, p.w_f32, p.w_vec, v * VEC, 0.f, b[i]);
    }
  }
  const float inv_c = 1.f / static_cast<float>(p.C);
  const long long step = static_cast<long long>(gridDim.x) * R;
  Vec<T, VEC> next[R][NV];
  auto fetch = [&](long long row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const T* row = static_cast<const T*>(p.x) + (row0 + r) * p.x_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i] && row0 + r < p.T) next[r][i].load(row + static_cast<size_t>(threadIdx.x + i * blockDim.x) * VEC);
    }
  };
  long long row0 = static_cast<long long>(blockIdx.x) * R;
  fetch(row0);
  for (; row0 < p.T; row0 += step) {
    float x[R][NV][VEC], s[R], mean[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        next[r][i].get(x[r][i]);
        if (has[i]) {  // (rows past the last hold what an earlier pass left there, and go nowhere)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[r] += x[r][i][e];
        }
      }
    }
    fetch(row0 + step);
    block_sum<R>(s, red[0]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      mean[r] = s[r] * inv_c;
      s[r] = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i]) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            x[r][i][e] -= mean[r];
            s[r] += x[r][i][e] * x[r][i][e];
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
      for (int i = 0; i < NV; ++i)
        if (has[i]) {
          float y[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = x[r][i][e] * rstd * w[i][e] + b[i][e];
          Vec<T, VEC>::put(out + static_cast<size_t>(threadIdx.x + i * blockDim.x) * VEC, y);
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
      load_param<T, 1>(p.w, p.w_f32, 0, c, 1.f, w);
      load_param<T, 1>(p.b, p.w_f32, 0, c, 0.f, b);
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
  __device__ __forceinline__ void get(float (&f)[VEC]) const { v.get(f); }
};
template <typename T, int VEC>
struct NormIn<T, VEC, true> {
  CodeVec<VEC> c;
  uint32_t scale;
  __device__ __forceinline__ void load(const NormParams& p, long long row, int vec) {
    const long long nb = pack_blocks(p.C);
    c.load(p.codes + row * nb * kPackBlock + static_cast<size_t>(vec) * VEC);
    scale = __ldg(p.scales + row * nb + vec * VEC / kPackBlock);
  }
  __device__ __forceinline__ void get(float (&f)[VEC]) const { c.get(pack_step(scale), f); }
};

template <typename T, int VEC, int NV, int R, bool PACKED>
__global__ void __launch_bounds__(R == 1 ? 1024 : R == 2 ? 512 : 256) layer_norm_bwd_kernel(const NormParams p) {
  __shared__ __align__(16) float red[2][2 * R * 32];
  const int nvec = p.C / VEC;
  float w[NV][VEC], dw[NV][VEC], db[NV][VEC];
  bool has[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    has[i] = v < nvec;
    if (has[i]) load_param<T, VEC>(p.w, p.w_f32, p.w_vec, v * VEC, 1.f, w[i]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) dw[i][e] = db[i][e] = 0.f;
  }
  const float inv_c = 1.f / static_cast<float>(p.C);
  const long long step = static_cast<long long>(gridDim.x) * R;
  NormIn<T, VEC, PACKED> nx[R][NV];
  Vec<T, VEC> ny[R][NV];
  float nmean[R], nrstd[R];
  auto fetch = [&](long long row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r;
      nmean[r] = nrstd[r] = 0.f;
      if (row < p.T) {
        nmean[r] = __ldg(p.mean + row);
        nrstd[r] = __ldg(p.rstd + row);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          const int v = threadIdx.x + i * blockDim.x;
          if (has[i]) {
            nx[r][i].load(p, row, v);
            ny[r][i].load(static_cast<const T*>(p.dy) + row * p.dy_stride + static_cast<size_t>(v) * VEC);
          }
        }
      }
    }
  };
  int phase = 0;
  long long row0 = static_cast<long long>(blockIdx.x) * R;
  fetch(row0);
  for (; row0 < p.T; row0 += step, phase ^= 1) {
    float h[R][NV][VEC], d[R][NV][VEC], rstd[R], s[2 * R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      s[2 * r] = s[2 * r + 1] = 0.f;
      rstd[r] = nrstd[r];
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i] && row0 + r < p.T) {
          nx[r][i].get(h[r][i]);
          ny[r][i].get(d[r][i]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float y = d[r][i][e], t = (h[r][i][e] - nmean[r]) * rstd[r], g = y * w[i][e];
            dw[i][e] += y * t;
            db[i][e] += y;
            s[2 * r] += g;
            s[2 * r + 1] += g * t;
            h[r][i][e] = t;
            d[r][i][e] = g;
          }
        }
    }
    fetch(row0 + step);
    block_sum<2 * R>(s, red[phase]);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r;
      if (row >= p.T) break;
      const float c1 = s[2 * r] * inv_c, c2 = s[2 * r + 1] * inv_c;
      T* out = static_cast<T*>(p.out) + row * p.out_stride;
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (has[i]) {
          float o[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[e] = rstd[r] * (d[r][i][e] - c1 - h[r][i][e] * c2);
          Vec<T, VEC>::put(out + static_cast<size_t>(threadIdx.x + i * blockDim.x) * VEC, o);
        }
    }
  }
  if (p.partial) {
    float* mine = p.partial + static_cast<size_t>(blockIdx.x) * 2 * p.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (has[i]) {
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
      load_param<T, 1>(p.w, p.w_f32, 0, c, 1.f, w);
      NormIn<T, 1, PACKED> in;
      float x[1];
      in.load(p, row, c);
      in.get(x);
      const float g = elem_f32<T>(dy[c]) * w[0];
      s[0] += g;
      s[1] += g * (x[0] - mean) * rstd;
    }
    block_sum<2>(s, red[phase]);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      float w[1];
      load_param<T, 1>(p.w, p.w_f32, 0, c, 1.f, w);
      NormIn<T, 1, PACKED> in;
      float x[1];
      in.load(p, row, c);
      in.get(x);
      out[c] = f32_elem<T>(rstd * (elem_f32<T>(dy[c]) * w[0] - c1 - (x[0] - mean) * rstd * c2));
    }
  }
}

template <typename T, bool PACKED>
__global__ void __launch_bounds__(256) layer_norm_bwd_wide_cols_kernel(const NormParams p) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= p.C) return;
  float dw = 0.f, db = 0.f;
  for (long long row = blockIdx.y; row < p.T; row += gridDim.y) {
    NormIn<T, 1, PACKED> in;
    float x[1];
    in.load(p, row, c);
    in.get(x);
    const float d = elem_f32<T>(static_cast<const T*>(p.dy)[row * p.dy_stride + c]);
    dw += d * (x[0] - __ldg(p.mean + row)) * __ldg(p.rstd + row);
    db += d;
  }
  p.partial[static_cast<size_t>(blockIdx.y) * 2 * p.C + c] = dw;
  p.partial[(static_cast<size_t>(blockIdx.y) * 2 + 1) * p.C + c] = db;
}

// out_a[c] = sum over g < groups of partial[g][a][c], a < arrays: 32 columns and
// 32 row lanes per block, the lanes' sums joined in a fixed order. Launched while the
// kernel that writes the partial rows still runs (programmatic dependent launch).
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
  float s = 0.f;
  if (c < p.C)
#pragma unroll 8
    for (int g = threadIdx.y; g < p.groups; g += 32)
      s += __ldcg(p.partial + (static_cast<size_t>(g) * p.arrays + a) * p.C + c);
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
      float f[VEC];
      x[r].get(f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        if (!has) f[e] = 0.f;
        m = max(m, abs_bits(f[e]));
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
      const uint32_t scale = pack_scale(m);
      const float inv = pack_inv(scale), lim = pack_limit(scale);
      if (in_row && row < p.T) {
        int8_t* dst = p.codes + row * nb * kPackBlock + static_cast<size_t>(v) * VEC;
        if constexpr (VEC == 1) {
          *dst = static_cast<int8_t>(pack_code(f[0], inv, lim));
        } else if constexpr (VEC == 4) {
          *reinterpret_cast<uint32_t*>(dst) = pack_code4(f[0], f[1], f[2], f[3], inv, lim);
        } else {
          *reinterpret_cast<uint2*>(dst) = make_uint2(pack_code4(f[0], f[1], f[2], f[3], inv, lim),
                                                      pack_code4(f[4], f[5], f[6], f[7], inv, lim));
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
        scale[r] = __ldg(p.scales + row * nb + v * VEC / kPackBlock);
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

// Rows of a block's pass: 4 for blocks of up to 256 threads, 2 up to 512 (registers),
// 1 for wider rows and where there are too few rows to give every SM a pass.
int rows_per_pass(int T, int threads) {
  const int r = threads <= 256 ? 4 : threads <= 512 ? 2 : 1;
  return T >= r * sms() ? r : 1;
}

// Blocks of a kernel that fit the GPU at once, at most one per pass. Per SM they are
// limited by registers; `cache` keeps the occupancy query's answer by warps per block.
template <typename K>
int resident_blocks(K kern, int threads, long long passes, int most_per_sm, signed char (&cache)[33]) {
  const int w = threads / 32;
  if (!cache[w]) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) != cudaSuccess || n < 1) n = 1;
    cache[w] = static_cast<signed char>(n);
  }
  const long long n = static_cast<long long>(sms()) * (cache[w] < most_per_sm ? cache[w] : most_per_sm);
  return static_cast<int>(passes < n ? passes : n);
}

// Partial rows of the weight gradients: at most this many blocks to an SM in the
// backward pass (each SM's loads stay in flight with fewer).
constexpr int kMaxBwdBlocksPerSm = 8;

template <typename T, int VEC, int NV, int R>
int launch_fwd(const NormParams& p, int threads, cudaStream_t st) {
  static signed char cache[33] = {0};
  auto kern = layer_norm_fwd_kernel<T, VEC, NV, R>;
  const int n = resident_blocks(kern, threads, (static_cast<long long>(p.T) + R - 1) / R, 32, cache);
  kern<<<n, threads, 0, st>>>(p);
  return launched();
}

template <typename T, int VEC, int NV, int R, bool PACKED>
int launch_bwd(const NormParams& p, int threads, int* groups, cudaStream_t st) {
  static signed char cache[33] = {0};
  auto kern = layer_norm_bwd_kernel<T, VEC, NV, R, PACKED>;
  *groups = resident_blocks(kern, threads, (static_cast<long long>(p.T) + R - 1) / R, kMaxBwdBlocksPerSm, cache);
  kern<<<*groups, threads, 0, st>>>(p);
  return launched();
}

template <typename T>
int norm_fwd(NormParams p, cudaStream_t st) {
  if (p.C > kMaxCols) {
    const int n = p.T < 2 * sms() ? p.T : 2 * sms();
    layer_norm_fwd_wide_kernel<T><<<n, 1024, 0, st>>>(p);
    return launched();
  }
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride).row(p.out, p.out_stride);
  p.w_vec = aligned_to(p.w, 16) && aligned_to(p.b, 16);
  return with_shape(rv.v, p.C, [&](auto vec, auto nv, int threads) {
    constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
    switch (rows_per_pass(p.T, threads)) {
      case 4: return launch_fwd<T, V, N, 4>(p, threads, st);
      case 2: return launch_fwd<T, V, N, 2>(p, threads, st);
      default: return launch_fwd<T, V, N, 1>(p, threads, st);
    }
  });
}

template <typename T, bool PACKED>
int norm_bwd(NormParams p, int* groups, cudaStream_t st) {
  if (p.C > kMaxCols) {
    const int n = p.T < 2 * sms() ? p.T : 2 * sms();
    layer_norm_bwd_wide_kernel<T, PACKED><<<n, 1024, 0, st>>>(p);
    if (p.partial) {
      *groups = p.T < sms() ? p.T : sms();
      layer_norm_bwd_wide_cols_kernel<T, PACKED><<<dim3((p.C + 255) / 256, *groups), 256, 0, st>>>(p);
    }
    return launched();
  }
  RowVec rv(p.C, sizeof(T));
  rv.row(p.x, p.x_stride).row(p.dy, p.dy_stride).row(p.out, p.out_stride);
  p.w_vec = aligned_to(p.w, 16);
  return with_shape(rv.v, p.C, [&](auto vec, auto nv, int threads) {
    constexpr int V = decltype(vec)::value, N = decltype(nv)::value;
    switch (rows_per_pass(p.T, threads)) {
      case 4: return launch_bwd<T, V, N, 4, PACKED>(p, threads, groups, st);
      case 2: return launch_bwd<T, V, N, 2, PACKED>(p, threads, groups, st);
      default: return launch_bwd<T, V, N, 1, PACKED>(p, threads, groups, st);
    }
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
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t lc = {};
  lc.gridDim = dim3((C + 31) / 32, arrays);
  lc.blockDim = dim3(32, 32);
  lc.stream = st;
  lc.attrs = &attr;
  lc.numAttrs = 1;
  if (cudaLaunchKernelEx(&lc, column_finish_kernel, f) != cudaSuccess) return FRATTN_E_CUDA;
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
  const long long blocks = static_cast<long long>(sms()) * kMaxBwdBlocksPerSm;
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
