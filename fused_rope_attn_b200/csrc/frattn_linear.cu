// Linear layer with bias, activation and residual in its epilogue, and its
// backward pass (sm_100a).
//
//   z = x W^T + b, out = act(z) + residual
//   dz = dout act'(z); dx = dz W, dw = dz^T x, db = sum over rows of dz
#include "frattn_block.cuh"

namespace frattn {

unsigned long long frattn_wait_limit_ns();  // frattn.cu
int column_finish(const float* partial, int groups, int arrays, int C, void* out0, void* out1, int dtype,
                  cudaStream_t st);  // frattn_norm.cu
int act_unpack(const int8_t* codes, const uint8_t* scales, int T, int C, int dtype, void* out, long long out_stride,
               cudaStream_t st);

// D[m, n] = sum_k A[m, k] B[n, k] with element strides, then the epilogue.
struct MatmulParams {
  const void *a, *b;
  long long a_m, a_k, b_n, b_k;
  int M, N, K;
  const void* bias;  // [N] or null
  const void* res;   // [M, N] or null
  long long res_stride;
  int act;
  void* out;
  long long out_stride;
  void* z;
  long long z_stride;
  int8_t* z_codes;
  uint8_t* z_scales;
};

namespace {

__device__ __forceinline__ float act_any(int act, float z) {
  switch (act) {
    case FRATTN_ACT_RELU: return act_f<FRATTN_ACT_RELU>(z);
    case FRATTN_ACT_GELU: return act_f<FRATTN_ACT_GELU>(z);
    case FRATTN_ACT_GELU_TANH: return act_f<FRATTN_ACT_GELU_TANH>(z);
    case FRATTN_ACT_SILU: return act_f<FRATTN_ACT_SILU>(z);
    default: return z;
  }
}

// 64 x 64 tile of D per block of 256 threads, 4 x 4 values per thread, fp32 FMAs.
template <typename T>
__global__ void __launch_bounds__(256) matmul_kernel(const MatmulParams p) {
  __shared__ float as[16][65], bs[16][65];
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int k = p.a_k == 1 ? i & 15 : i >> 6, m = p.a_k == 1 ? i >> 4 : i & 63;
      as[k][m] = m0 + m < p.M && k0 + k < p.K
                     ? elem_f32<T>(static_cast<const T*>(p.a)[(m0 + m) * p.a_m + (k0 + k) * p.a_k]) : 0.f;
      const int kb = p.b_k == 1 ? i & 15 : i >> 6, n = p.b_k == 1 ? i >> 4 : i & 63;
      bs[kb][n] = n0 + n < p.N && k0 + kb < p.K
                      ? elem_f32<T>(static_cast<const T*>(p.b)[(n0 + n) * p.b_n + (k0 + kb) * p.b_k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      float a[4], b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = as[k][ty * 4 + i];
        b[i] = bs[k][tx * 4 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] += a[i] * b[j];
    }
    __syncthreads();
  }
  const int nb = static_cast<int>(pack_blocks(p.N));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + ty * 4 + i;
    uint32_t amax = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n < p.N && p.bias) acc[i][j] += elem_f32<T>(static_cast<const T*>(p.bias)[n]);
      if (n < p.N) amax = max(amax, abs_bits(acc[i][j]));
    }
    if (p.z_codes) {  // 8 neighbouring threads hold a block of 32 columns
#pragma unroll
      for (int o = 4; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const uint32_t scale = pack_scale(amax);
      const float inv = pack_inv(scale);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int n = n0 + tx * 4 + j;
        if (m < p.M && n < nb * kPackBlock)
          p.z_codes[m * nb * kPackBlock + n] = n < p.N ? static_cast<int8_t>(pack_code(acc[i][j], inv)) : 0;
      }
      if (m < p.M && (tx & 7) == 0 && n0 + tx * 4 < p.N)
        p.z_scales[m * nb + (n0 + tx * 4) / kPackBlock] = static_cast<uint8_t>(scale);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      if (p.z) static_cast<T*>(p.z)[m * p.z_stride + n] = f32_elem<T>(acc[i][j]);
      float y = act_any(p.act, acc[i][j]);
      if (p.res) y += elem_f32<T>(static_cast<const T*>(p.res)[m * p.res_stride + n]);
      static_cast<T*>(p.out)[m * p.out_stride + n] = f32_elem<T>(y);
    }
  }
}

template <typename T>
int matmul(const MatmulParams& p, cudaStream_t st) {
  matmul_kernel<T><<<dim3((p.N + 63) / 64, (p.M + 63) / 64), 256, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : FRATTN_E_CUDA;
}

// dz = dout act'(z) over rows of N columns, with partial column sums of dz.
struct ActBwdParams {
  const void* dout;
  long long dout_stride;
  const void* z;
  long long z_stride;
  const int8_t* z_codes;
  const uint8_t* z_scales;
  void* dz;  // null: column sums only
  long long dz_stride;
  float* partial;  // [gridDim.y][N] or null
  int T, N;
};

// One thread owns VEC columns over a strip of rows (rows blockIdx.y,
// blockIdx.y + gridDim.y, ...): neighbouring threads read neighbouring vectors,
// the column sums stay in registers, R rows are in flight at a time.
template <typename T, int VEC, int ACT, bool PACKED>
__global__ void __launch_bounds__(256) act_bwd_kernel(const ActBwdParams p) {
  constexpr int R = 4;
  const int v = blockIdx.x * blockDim.x + threadIdx.x;
  if (v * VEC >= p.N) return;
  const size_t c = static_cast<size_t>(v) * VEC;
  const int nb = static_cast<int>(pack_blocks(p.N));
  float sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
  const long long step = gridDim.y;
  for (long long row0 = blockIdx.y; row0 < p.T; row0 += step * R) {
    Vec<T, VEC> dy[R], z[R];
    union {
      typename RawVec<VEC == 1 ? 2 : VEC>::type raw;
      int8_t c[VEC == 1 ? 2 : VEC];
    } q[R];
    uint32_t scale[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row < p.T) {
        dy[r].load(static_cast<const T*>(p.dout) + row * p.dout_stride + c);
        if constexpr (ACT != FRATTN_ACT_NONE) {
          if constexpr (PACKED) {
            const int8_t* src = p.z_codes + row * nb * kPackBlock + c;
            if constexpr (VEC == 1) q[r].c[0] = __ldg(src);
            else q[r].raw = __ldg(reinterpret_cast<const typename RawVec<VEC>::type*>(src));
            scale[r] = __ldg(p.z_scales + row * nb + v * VEC / kPackBlock);
          } else {
            z[r].load(static_cast<const T*>(p.z) + row * p.z_stride + c);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row >= p.T) break;
      const float st = PACKED && ACT != FRATTN_ACT_NONE ? pack_step(scale[r]) : 0.f;
      Vec<T, VEC> o;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        float d = dy[r].get(e);
        if constexpr (ACT != FRATTN_ACT_NONE)
          d *= act_grad_f<ACT>(PACKED ? static_cast<float>(q[r].c[e]) * st : z[r].get(e));
        sum[e] += d;
        o.set(e, d);
      }
      if (p.dz) o.store(static_cast<T*>(p.dz) + row * p.dz_stride + c);
    }
  }
  if (p.partial) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.partial[static_cast<size_t>(blockIdx.y) * p.N + c + e] = sum[e];
  }
}

constexpr int kMaxStrips = 592;  // partial rows of the bias gradient

template <typename T, int VEC, int ACT, bool PACKED>
int act_bwd_launch(const ActBwdParams& p, int* groups, cudaStream_t st) {
  const int nv = p.N / VEC;
  const int tiles = (nv + 255) / 256;
  const int bx = ((nv + tiles - 1) / tiles + 31) / 32 * 32;
  const int gx = (nv + bx - 1) / bx;
  long long gy = static_cast<long long>(sm_count_for_current_device()) * 8 / gx;
  const long long rows4 = (p.T + 3) / 4;
  if (gy > rows4) gy = rows4;
  if (gy > kMaxStrips) gy = kMaxStrips;
  if (gy < 1) gy = 1;
  *groups = static_cast<int>(gy);
  act_bwd_kernel<T, VEC, ACT, PACKED><<<dim3(gx, static_cast<unsigned>(gy)), bx, 0, st>>>(p);
  return cudaGetLastError() == cudaSuccess ? 0 : FRATTN_E_CUDA;
}

template <typename T, int VEC, bool PACKED>
int act_bwd_act(const ActBwdParams& p, int act, int* groups, cudaStream_t st) {
  switch (act) {
    case FRATTN_ACT_RELU: return act_bwd_launch<T, VEC, FRATTN_ACT_RELU, PACKED>(p, groups, st);
    case FRATTN_ACT_GELU: return act_bwd_launch<T, VEC, FRATTN_ACT_GELU, PACKED>(p, groups, st);
    case FRATTN_ACT_GELU_TANH: return act_bwd_launch<T, VEC, FRATTN_ACT_GELU_TANH, PACKED>(p, groups, st);
    case FRATTN_ACT_SILU: return act_bwd_launch<T, VEC, FRATTN_ACT_SILU, PACKED>(p, groups, st);
    default: return act_bwd_launch<T, VEC, FRATTN_ACT_NONE, false>(p, groups, st);
  }
}

template <typename T>
int act_bwd(const ActBwdParams& p, int act, int* groups, cudaStream_t st) {
  RowVec rv(p.N, sizeof(T));
  rv.row(p.dout, p.dout_stride).row(p.z, p.z_stride).row(p.dz, p.dz_stride);
  if (rv.v == 8) return p.z_codes ? act_bwd_act<T, 8, true>(p, act, groups, st) : act_bwd_act<T, 8, false>(p, act, groups, st);
  if (rv.v == 4) return p.z_codes ? act_bwd_act<T, 4, true>(p, act, groups, st) : act_bwd_act<T, 4, false>(p, act, groups, st);
  return p.z_codes ? act_bwd_act<T, 1, true>(p, act, groups, st) : act_bwd_act<T, 1, false>(p, act, groups, st);
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

// Workspace of the backward pass: dz [T, Np] (rows padded to 16 bytes), partial
// column sums, and the 16-bit values of a packed x [T, Kp].
struct BwdLayout {
  long long np, kp;
  size_t dz, partial, x, total;
};
BwdLayout bwd_layout(int T, int K, int N) {
  BwdLayout l;
  l.np = (static_cast<long long>(N) + 7) / 8 * 8;
  l.kp = (static_cast<long long>(K) + 7) / 8 * 8;
  l.dz = 0;
  l.partial = up256(static_cast<size_t>(T) * l.np * 2);
  l.x = l.partial + up256(static_cast<size_t>(kMaxStrips) * N * sizeof(float));
  l.total = l.x + up256(static_cast<size_t>(T) * l.kp * 2);
  return l;
}

template <typename T>
int linear_bwd(const void* dout, long long dout_stride, const void* x, long long x_stride, const int8_t* x_codes,
               const uint8_t* x_scales, const void* w, long long w_stride, const void* z, long long z_stride,
               const int8_t* z_codes, const uint8_t* z_scales, int act, int rows, int K, int N, int dtype, void* dx,
               long long dx_stride, void* dw, void* db, uint8_t* ws, cudaStream_t st) {
  const BwdLayout l = bwd_layout(rows, K, N);
  const bool in_place = act == FRATTN_ACT_NONE && aligned_to(dout, 16) && dout_stride % 8 == 0;
  const void* dz = in_place ? dout : ws + l.dz;
  const long long dz_stride = in_place ? dout_stride : l.np;
  int rc = 0;
  if (!in_place || db) {
    ActBwdParams a;
    memset(&a, 0, sizeof(a));
    a.dout = dout;
    a.dout_stride = dout_stride;
    if (act != FRATTN_ACT_NONE) {
      a.z = z;
      a.z_stride = z_stride;
      a.z_codes = z_codes;
      a.z_scales = z_scales;
    }
    a.dz = in_place ? nullptr : ws + l.dz;
    a.dz_stride = l.np;
    a.partial = db ? reinterpret_cast<float*>(ws + l.partial) : nullptr;
    a.T = rows;
    a.N = N;
    int groups = 0;
    if (rows > 0 && (rc = act_bwd<T>(a, act, &groups, st))) return rc;
    if (db && (rc = column_finish(reinterpret_cast<float*>(ws + l.partial), groups, 1, N, db, nullptr, dtype, st)))
      return rc;
  }
  MatmulParams m;
  if (dx && rows > 0) {
    memset(&m, 0, sizeof(m));
    m.a = dz;
    m.a_m = dz_stride;
    m.a_k = 1;
    m.b = w;
    m.b_n = 1;
    m.b_k = w_stride;
    m.M = rows;
    m.N = K;
    m.K = N;
    m.out = dx;
    m.out_stride = dx_stride;
    if ((rc = matmul<T>(m, st))) return rc;
  }
  if (dw) {
    if (x_codes && rows > 0) {
      if ((rc = act_unpack(x_codes, x_scales, rows, K, dtype, ws + l.x, l.kp, st))) return rc;
      x = ws + l.x;
      x_stride = l.kp;
    }
    memset(&m, 0, sizeof(m));
    m.a = dz;
    m.a_m = 1;
    m.a_k = dz_stride;
    m.b = x;
    m.b_n = 1;
    m.b_k = x_stride;
    m.M = N;
    m.N = K;
    m.K = rows;
    m.out = dw;
    m.out_stride = K;
    if ((rc = matmul<T>(m, st))) return rc;
  }
  return 0;
}

bool rows16(const void* p, long long stride) { return aligned_to(p, 16) && stride % 8 == 0; }

}  // namespace
}  // namespace frattn

using namespace frattn;

extern "C" {

int frattn_workspace_bytes_linear_act(int T, int K, int N, size_t* bytes) {
  if (!bytes) return FRATTN_E_NULL;
  if (T < 0 || K <= 0 || N <= 0) return FRATTN_E_SHAPE;
  *bytes = 0;
  return 0;
}

int frattn_linear_act(const void* x, long long x_stride, const void* w, long long w_stride, const void* bias,
                      const void* residual, long long res_stride, int activation, int T, int K, int N, int dtype,
                      void* out, long long out_stride, void* z, long long z_stride, int8_t* z_codes,
                      uint8_t* z_scales, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (T < 0 || K <= 0 || N <= 0 || x_stride < K || w_stride < K || out_stride < N || (residual && res_stride < 0) ||
      (z && z_stride < N) || activation < FRATTN_ACT_NONE || activation > FRATTN_ACT_SILU)
    return FRATTN_E_SHAPE;
  if (dtype != FRATTN_BF16 && dtype != FRATTN_F16) return FRATTN_E_DTYPE;
  if (T == 0) return 0;
  if (!x || !w || !out || (z && z_codes) || !z_codes != !z_scales) return FRATTN_E_NULL;
  if (!rows16(x, x_stride) || !rows16(w, w_stride) || !aligned_to(bias, 2) || !aligned_to(residual, 2) ||
      !aligned_to(out, 2) || !aligned_to(z, 2) || !aligned_to(z_codes, 16))
    return FRATTN_E_ALIGN;
  size_t need = 0;
  frattn_workspace_bytes_linear_act(T, K, N, &need);
  if (workspace_bytes < need) return FRATTN_E_WORKSPACE;
  (void)workspace;
  (void)status;
  MatmulParams m;
  memset(&m, 0, sizeof(m));
  m.a = x;
  m.a_m = x_stride;
  m.a_k = 1;
  m.b = w;
  m.b_n = w_stride;
  m.b_k = 1;
  m.M = T;
  m.N = N;
  m.K = K;
  m.bias = bias;
  m.res = residual;
  m.res_stride = res_stride;
  m.act = activation;
  m.out = out;
  m.out_stride = out_stride;
  m.z = z;
  m.z_stride = z_stride;
  m.z_codes = z_codes;
  m.z_scales = z_scales;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == FRATTN_BF16 ? matmul<__nv_bfloat16>(m, st) : matmul<__half>(m, st);
}

int frattn_workspace_bytes_linear_act_bwd(int T, int K, int N, size_t* bytes) {
  if (!bytes) return FRATTN_E_NULL;
  if (T < 0 || K <= 0 || N <= 0) return FRATTN_E_SHAPE;
  *bytes = bwd_layout(T, K, N).total;
  return 0;
}

int frattn_linear_act_bwd(const void* dout, long long dout_stride, const void* x, long long x_stride,
                          const int8_t* x_codes, const uint8_t* x_scales, const void* w, long long w_stride,
                          const void* z, long long z_stride, const int8_t* z_codes, const uint8_t* z_scales,
                          int activation, int T, int K, int N, int dtype, void* dx, long long dx_stride, void* dw,
                          void* db, void* workspace, size_t workspace_bytes, int32_t* status, void* stream) {
  if (T < 0 || K <= 0 || N <= 0 || dout_stride < 0 || (x && x_stride < K) || (dx && w_stride < K) ||
      (z && z_stride < 0) || (dx && dx_stride < K) || activation < FRATTN_ACT_NONE || activation > FRATTN_ACT_SILU)
    return FRATTN_E_SHAPE;
  if (dtype != FRATTN_BF16 && dtype != FRATTN_F16) return FRATTN_E_DTYPE;
  if (!workspace) return FRATTN_E_NULL;
  if (T > 0) {
    if (!dout || (dx && !w)) return FRATTN_E_NULL;
    if (dw && (x ? x_codes || x_scales : !x_codes || !x_scales)) return FRATTN_E_NULL;
    if (activation != FRATTN_ACT_NONE && (z ? z_codes || z_scales : !z_codes || !z_scales)) return FRATTN_E_NULL;
  }
  if (!aligned_to(dout, 2) || (dw && x && !rows16(x, x_stride)) || (dx && !rows16(w, w_stride)) ||
      !aligned_to(z, 2) || !aligned_to(dx, 2) || !aligned_to(dw, 2) || !aligned_to(db, 2) ||
      !aligned_to(x_codes, 16) || !aligned_to(z_codes, 16) || !aligned_to(workspace, 256))
    return FRATTN_E_ALIGN;
  size_t need = 0;
  frattn_workspace_bytes_linear_act_bwd(T, K, N, &need);
  if (workspace_bytes < need) return FRATTN_E_WORKSPACE;
  (void)status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (dtype == FRATTN_BF16)
    return linear_bwd<__nv_bfloat16>(dout, dout_stride, x, x_stride, x_codes, x_scales, w, w_stride, z, z_stride,
                                     z_codes, z_scales, activation, T, K, N, dtype, dx, dx_stride, dw, db, ws, st);
  return linear_bwd<__half>(dout, dout_stride, x, x_stride, x_codes, x_scales, w, w_stride, z, z_stride, z_codes,
                            z_scales, activation, T, K, N, dtype, dx, dx_stride, dw, db, ws, st);
}

}  // extern "C"
