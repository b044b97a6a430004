// Linear layer with bias, activation and residual in its epilogue, and its
// backward pass (sm_100a).
//
//   z = x W^T + b, out = act(z) + residual
//   dz = dout act'(z); dx = dz W, dw = dz^T x, db = sum over rows of dz
//
// Three products on the tensor cores (tcgen05, fp32 sums in TMEM), all through TMA with
// 128-byte swizzle; the backward's operands that run along m or n instead of along the
// reduction are read as they lie in memory, MN-major, with no transposed copies. Large
// products run on CTA pairs (gemm_pair_kernel), small ones on clusters that split the
// reduction (gemm_small_kernel). dz and db come from one pass over dout and z
// (act_bwd_kernel); dz is rounded to 16 bits once, since the tensor cores take it so.
//
// Measured, bf16, kernels alone: 9216 x 1280 -> 3424 in 65 us (1.24 PFLOP/s; cuBLAS's
// bare product 61), with gelu 75, with a packed pre-activation too 82; 9216 x 3424 ->
// 1280 with residual 71; the main loop alone takes 55 and 62. The backward of 9216 x
// 1280 -> 3424 with gelu_tanh takes 172 us: dz and db about 44, dx 66, dw 62. Run for
// longer than some milliseconds these are bound by the card's power (cuBLAS's 61 us
// become 73, 71 and 172 here become 83 and 200), so that every instruction of the
// epilogue shows, hidden or not.
#include "frattn_block.cuh"

namespace frattn {

unsigned long long frattn_wait_limit_ns();  // frattn.cu
int column_finish(const float* partial, int groups, int arrays, int C, void* out0, void* out1, int dtype,
                  cudaStream_t st);  // frattn_norm.cu
int act_unpack(const int8_t* codes, const uint8_t* scales, int T, int C, int dtype, void* out, long long out_stride,
               cudaStream_t st);

// One product D[m, n] = sum_k A[m, k] B[n, k] and its epilogue. A and B are matrices of
// 16-bit rows; an operand is "K-major" when its rows run along k (x and W in the
// forward product), "MN-major" when they run along m or n (W in dz W, both in dz^T x).
struct GemmParams {
  CUtensorMap tma_a, tma_b;
  CUtensorMap tma_out, tma_z, tma_res;  // box {64, 32}, 128-byte swizzle; used where *_tma
  CUtensorMap tma_codes;                // box {64, 32} bytes, 64-byte swizzle
  const void* bias;            // [N] or null
  const void* res;             // [M, N] or null
  long long res_stride;
  int act;
  void* out;
  long long out_stride;
  void* z;  // or null
  long long z_stride;
  int8_t* z_codes;  // or null
  uint8_t* z_scales;
  int out_tma, z_tma;          // written by TMA stores (16-byte rows; the pair kernel)
  int out_w, z_w;              // else elements per store: 8 (where N allows it), 4, 2 or 1
  int res_tma;                 // residual read ahead by TMA (16-byte rows, nothing else staged)
  int res_vec;                 // residual rows are 16-byte aligned
  int M, N, nk;                // nk: 64-wide steps of the reduction
  int a_bytes;                 // of A in a stage (small products)
  int tiles_n, tiles;
  int split;                   // 0: a pair owns whole tiles; else k steps per pair (see Segments)
  float* partial;              // [2 pairs][BN / 4][256][4] (split)
  int32_t* status;
  unsigned long long wait_limit_ns;
};

namespace {

template <int BN>
struct GemmCfg {
  static constexpr int BK = 64;
  static constexpr int A_BYTES = 128 * BK * 2;
  static constexpr int B_BYTES = BN / 2 * BK * 2;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int EPI_WARPS = 4 * ((BN + 63) / 64);  // four lane quarters x 64-column chunks
  static constexpr int THREADS = 64 + 32 * EPI_WARPS;      // warp 0 TMA, warp 1 MMA, the rest epilogue
  static constexpr int STG = 32 * 64 * 2;                  // a warp's staging: 32 rows x 64 columns of 16 bits
  static constexpr int STG_BYTES = EPI_WARPS * STG;
  static constexpr int BIAS_BYTES = EPI_WARPS * 64 * 4;
  static constexpr int ST_FIT = (227 * 1024 - 1024 - 512 - STG_BYTES - BIAS_BYTES) / STAGE;
  static constexpr int ST = ST_FIT > 8 ? 8 : ST_FIT;
  static constexpr int OFF_STG = ST * STAGE;
  static constexpr int OFF_BIAS = OFF_STG + STG_BYTES;
  static constexpr int OFF_BAR = OFF_BIAS + BIAS_BYTES;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;  // barriers + 1024-B alignment slack
  static_assert(STAGE % 1024 == 0 && OFF_STG % 1024 == 0, "128-B swizzle atoms");
  static_assert((2 * ST + 5 + EPI_WARPS) * 8 + 8 <= 512, "barriers");
};

// The tiles (or parts of tiles) a CTA pair computes, in order; every role of the
// kernel walks the same list.
//  * whole tiles: t = pair, pair + pairs, ... with all nk steps each;
//  * split: the nk steps of all tiles, laid end to end, are dealt out in equal runs
//    of `split` steps. A pair's run covers at most one part at the end of a tile
//    that an earlier pair began, whole tiles, and one part at the beginning of a
//    tile that it does not finish. Parts go to the pair's two partial slots as
//    fp32 sums; gemm_finish_kernel adds a tile's parts in the order of k.
struct Segments {
  int t, k0, k1;
  int pos, end, step, split, nk, tiles;
  __device__ __forceinline__ Segments(const GemmParams& p, int pair, int pairs) {
    split = p.split;
    nk = p.nk;
    tiles = p.tiles;
    if (split) {
      const long long total = static_cast<long long>(tiles) * nk;
      const long long b = static_cast<long long>(pair) * split;
      pos = static_cast<int>(b < total ? b : total);
      end = static_cast<int>(b + split < total ? b + split : total);
      step = 0;
    } else {
      pos = pair;
      end = tiles;
      step = pairs;
    }
  }
  __device__ __forceinline__ bool next() {
    if (pos >= end) return false;
    if (split) {
      t = pos / nk;
      k0 = pos - t * nk;
      const int room = end - pos;
      k1 = nk - k0 < room ? nk : k0 + room;
      pos += k1 - k0;
    } else {
      t = pos;
      k0 = 0;
      k1 = nk;
      pos += step;
    }
    return true;
  }
  __device__ __forceinline__ bool whole() const { return k0 == 0 && k1 == nk; }
};

__device__ __forceinline__ bool gemm_wait(uint32_t bar, uint32_t parity, const GemmParams& p,
                                          volatile int* abort_flag, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t n = 0;
  while (!mbar_try_wait(bar, parity)) {
    if ((++n & 15u) == 0) {
      if (*abort_flag) return false;
      if (globaltimer_ns() - t0 > p.wait_limit_ns) {
        *abort_flag = 1;
        if (p.status) atomicCAS(reinterpret_cast<int*>(p.status), 0, code);
        return false;
      }
    }
  }
  return true;
}

// Drain wait used while unwinding: ignores the abort flag, gives up after limit.
__device__ __forceinline__ void gemm_drain(uint32_t bar, uint32_t parity, unsigned long long limit) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > limit) return;
}

template <int ACT, int N>
__device__ __forceinline__ void act_all(float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) act_f2<ACT>(v[i], v[i + 1]);
}
template <int N>
__device__ __forceinline__ void act_any(int act, float (&v)[N]) {
  switch (act) {
    case FRATTN_ACT_RELU: return act_all<FRATTN_ACT_RELU>(v);
    case FRATTN_ACT_GELU: return act_all<FRATTN_ACT_GELU>(v);
    case FRATTN_ACT_GELU_TANH: return act_all<FRATTN_ACT_GELU_TANH>(v);
    case FRATTN_ACT_SILU: return act_all<FRATTN_ACT_SILU>(v);
    default: return;
  }
}

// A warp's staging holds 32 rows of 64 columns (16 bits: 128 bytes a row, 128-byte
// swizzle) as the TMA transfers expect it: 16-byte part c of row r lies at c ^ (r & 7),
// which also spreads the lanes over the banks.
__device__ __forceinline__ uint4* stage_part(uint8_t* stg, int r, int c) {
  return reinterpret_cast<uint4*>(stg + r * 128 + ((c ^ (r & 7)) << 4));
}
// 32 values of row r into the staging's columns [32 h, 32 h + 32).
template <typename T>
__device__ __forceinline__ void stage32(uint8_t* stg, int r, int h, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint4 w;
    w.x = pack2<T>(v[8 * c + 0], v[8 * c + 1]);
    w.y = pack2<T>(v[8 * c + 2], v[8 * c + 3]);
    w.z = pack2<T>(v[8 * c + 4], v[8 * c + 5]);
    w.w = pack2<T>(v[8 * c + 6], v[8 * c + 7]);
    *stage_part(stg, r, 4 * h + c) = w;
  }
}

// The warp writes its staging, rows [m, m + 32) and columns [n, n + 64), to a matrix
// whose rows are not 16-byte aligned: W elements per lane, a row's in neighbouring lanes.
template <int W>
__device__ __forceinline__ void store_rows_w(const uint8_t* stg, int lane, void* out, long long stride, long long m,
                                             int n, int M, int N) {
  using Raw = typename RawVec<2 * W>::type;
  constexpr int LANES = 64 / W;  // lanes of a row
#pragma unroll 4
  for (int i = lane; i < 32 * LANES; i += 32) {
    const int r = i / LANES, c = i % LANES * W;
    if (m + r < M && n + c < N)  // (W divides N: a vector lies inside the row or outside)
      *reinterpret_cast<Raw*>(static_cast<uint16_t*>(out) + (m + r) * stride + n + c) =
          *reinterpret_cast<const Raw*>(stg + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
  }
}
// The staged 16-bit values to a matrix, by TMA where its rows allow.
__device__ __forceinline__ void store_staged(const CUtensorMap* map, int tma, int width, uint8_t* stg, int lane, void* out,
                                             long long stride, int m0, int n0, int M, int N) {
  if (tma) {
    fence_proxy_async_smem();  // the warp's staging writes, visible to the TMA store
    __syncwarp();
    if (lane == 0) {
      tma_store_2d(map, smem_u32(stg), n0, m0);
      bulk_commit_group();
    }
  } else {
    __syncwarp();
    if (width >= 4) store_rows_w<4>(stg, lane, out, stride, m0, n0, M, N);
    else if (width == 2) store_rows_w<2>(stg, lane, out, stride, m0, n0, M, N);
    else store_rows_w<1>(stg, lane, out, stride, m0, n0, M, N);
    __syncwarp();
  }
}
// Lane 0's TMA stores have read the staging: the warp may write it again.
__device__ __forceinline__ void staging_free(int lane) {
  if (lane == 0) bulk_wait_read_all();
  __syncwarp();
}

__device__ __forceinline__ void add_bias(float (&v)[32], const float* bias) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 b = reinterpret_cast<const float4*>(bias)[i];
    v[4 * i] += b.x;
    v[4 * i + 1] += b.y;
    v[4 * i + 2] += b.z;
    v[4 * i + 3] += b.w;
  }
}

// The epilogue of a warp's piece of D, rows [m, m + 32) (one a lane) and columns
// [n, n + 32), of which v holds the lane's row (columns past N hold zeros). `stg`: 2 KB of
// the warp's own, through which rows are written a row's parts in neighbouring lanes
// (16-byte part c of row r at c ^ (r / 2 & 3), 64-byte rows).
template <typename T, int W>
__device__ __forceinline__ void put_piece_w(const uint8_t* stg, int lane, void* out, long long stride, long long m, int n,
                                            int M, int N) {
  using Raw = typename RawVec<2 * W>::type;
  constexpr int LANES = 32 / W;  // lanes of a row
#pragma unroll 8
  for (int i = lane; i < 32 * LANES; i += 32) {
    const int r = i / LANES, c = i % LANES * W;
    if (m + r < M && n + c < N)  // (W divides N: a vector lies inside the row or outside)
      *reinterpret_cast<Raw*>(static_cast<uint16_t*>(out) + (m + r) * stride + n + c) =
          *reinterpret_cast<const Raw*>(stg + r * 64 + (((c >> 3) ^ ((r >> 1) & 3)) << 4) + (c & 7) * 2);
  }
}
template <typename T>
__device__ __forceinline__ void put_piece(uint8_t* stg, int lane, void* out, long long stride, long long m, int n, int M,
                                          int N, int width, const float (&v)[32]) {
  __syncwarp();
#pragma unroll
  for (int c = 0; c < 4; ++c)
    *reinterpret_cast<uint4*>(stg + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(pack2<T>(v[8 * c], v[8 * c + 1]), pack2<T>(v[8 * c + 2], v[8 * c + 3]),
                   pack2<T>(v[8 * c + 4], v[8 * c + 5]), pack2<T>(v[8 * c + 6], v[8 * c + 7]));
  __syncwarp();
  if (width == 8) put_piece_w<T, 8>(stg, lane, out, stride, m, n, M, N);
  else if (width == 4) put_piece_w<T, 4>(stg, lane, out, stride, m, n, M, N);
  else if (width == 2) put_piece_w<T, 2>(stg, lane, out, stride, m, n, M, N);
  else put_piece_w<T, 1>(stg, lane, out, stride, m, n, M, N);
}
template <typename T>
__device__ __forceinline__ void finish_piece(const GemmParams& p, long long m, int n, int lane, uint8_t* stg, float (&v)[32]) {
  const long long row = m + lane;
  if (p.bias) {
    const float b = n + lane < p.N ? elem_f32<T>(static_cast<const T*>(p.bias)[n + lane]) : 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += __shfl_sync(0xffffffffu, b, i);
  }
  if (p.z) put_piece<T>(stg, lane, p.z, p.z_stride, m, n, p.M, p.N, p.z_w, v);
  if (p.z_codes && row < p.M) {
    const long long nb = pack_blocks(p.N);
    uint32_t codes[8];
    p.z_scales[row * nb + n / 32] = static_cast<uint8_t>(pack32(v, codes));
#pragma unroll
    for (int c = 0; c < 2; ++c)
      reinterpret_cast<uint4*>(p.z_codes + (row * nb + n / 32) * kPackBlock)[c] =
          make_uint4(codes[4 * c], codes[4 * c + 1], codes[4 * c + 2], codes[4 * c + 3]);
  }
  act_any(p.act, v);
  if (p.res && row < p.M) {
    const T* rp = static_cast<const T*>(p.res) + row * p.res_stride + n;
    if (p.res_vec && n + 32 <= p.N) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float f[8];
        unpack8<T>(reinterpret_cast<const uint4*>(rp)[c], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * c + e] += f[e];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (n + i < p.N) v[i] += elem_f32<T>(rp[i]);
    }
  }
  put_piece<T>(stg, lane, p.out, p.out_stride, m, n, p.M, p.N, p.out_w, v);
}

// GEMM on CTA pairs (cluster of 2, tcgen05 cta_group::2): 256 x BN tiles of D, M = 256
// MMAs spanning both CTAs, each CTA loading its 128 rows of A and half of the B tile by
// TMA (128-byte swizzle) into an ST-stage ring, fp32 accumulators in TMEM (two of BN
// columns: the epilogue of a tile runs under the main loop of the next). The epilogue
// warps each take 64 columns of a TMEM lane quarter, 32 values of a row per thread and
// step, so a block of 32 of a packed pre-activation is one thread's. (Sixteen warps: with
// eight of them the epilogue, not the main loop, set the pace of K = 1280 with gelu:
// two warps to a scheduler leave most of its issue slots empty.) Waits are bounded; on a
// timeout the kernel records a status code, waits (bounded) for its own copies and MMAs,
// frees TMEM and returns.
template <int BN, bool AMN, bool BMN, typename T>
__global__ void __launch_bounds__(GemmCfg<BN>::THREADS, 1) gemm_pair_kernel(const __grid_constant__ GemmParams p) {
  using C = GemmCfg<BN>;
  constexpr int ST = C::ST;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC = make_idesc_f16(kBF16, 256, BN, BMN) | (AMN ? 1u << 15 : 0u);
  constexpr uint32_t SW128 = 2;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int FULL = 0, EMPTY = ST, ACC_FULL = 2 * ST, ACC_EMPTY = 2 * ST + 2, DRAIN = 2 * ST + 4;
  const int RES = 2 * ST + 5;  // residual chunk of each epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * ST + 5 + C::EPI_WARPS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(bar(FULL + i), 1);   // the leader's producer arrives; both CTAs' bytes complete it
      mbar_init(bar(EMPTY + i), 1);  // multicast commit of the leader's MMAs
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ACC_FULL + i), 1);
      mbar_init(bar(ACC_EMPTY + i), 2 * C::EPI_WARPS);  // epilogue warps of both CTAs (used in the leader)
    }
    mbar_init(bar(DRAIN), 1);
    for (int i = 0; i < C::EPI_WARPS; ++i) mbar_init(bar(RES + i), 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tma_a);
    tma_prefetch_desc(&p.tma_b);
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();  // barriers of both CTAs initialised, TMEM allocated
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------------------------------------------------- producer (both CTAs)
      uint32_t it = 0;
      bool ok = true;
      for (Segments s(p, pair, pairs); ok && s.next();) {
        const int m0 = (s.t / p.tiles_n) * 256 + 128 * static_cast<int>(rank);
        const int n0 = (s.t % p.tiles_n) * BN + BN / 2 * static_cast<int>(rank);
        for (int kb = s.k0; kb < s.k1; ++kb, ++it) {
          const int st = it % ST;
          if (!gemm_wait(bar(EMPTY + st), ((it / ST) & 1) ^ 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x71)) {
            ok = false;
            break;
          }
          if (leader) mbar_arrive_expect_tx(bar(FULL + st), 2 * C::STAGE);
          const uint32_t full0 = mapa_shared(bar(FULL + st), 0);  // the leader's stage barrier
          const uint32_t a = smem_u32(smem + st * C::STAGE), b = a + C::A_BYTES;
          if constexpr (AMN) {  // two boxes of 64 columns x 64 rows of the reduction
            tma_load_2d_pair(a, &p.tma_a, full0, m0, kb * C::BK);
            tma_load_2d_pair(a + 8192, &p.tma_a, full0, m0 + 64, kb * C::BK);
          } else {
            tma_load_2d_pair(a, &p.tma_a, full0, kb * C::BK, m0);
          }
          if constexpr (BMN) {
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)
              tma_load_2d_pair(b + 8192 * j, &p.tma_b, full0, n0 + 64 * j, kb * C::BK);
          } else {
            tma_load_2d_pair(b, &p.tma_b, full0, kb * C::BK, n0);
          }
        }
      }
      if (leader) {  // copies of both CTAs still in flight land before the pair exits
        const uint32_t first = it > static_cast<uint32_t>(ST) ? it - ST : 0;
        for (uint32_t i = first; i < it; ++i) gemm_drain(bar(FULL + i % ST), (i / ST) & 1, p.wait_limit_ns);
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ---------------------------------------------------------- MMA issuer (leader)
      uint32_t it = 0, lt = 0;
      bool ok = true;
      for (Segments s(p, pair, pairs); ok && s.next(); ++lt) {
        const int buf = lt & 1;
        if (!gemm_wait(bar(ACC_EMPTY + buf), ((lt >> 1) & 1) ^ 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x72))
          break;
        tc_fence_after();
        const uint32_t d = tmem + buf * 256u;
        for (int kb = s.k0; kb < s.k1; ++kb, ++it) {
          const int st = it % ST;
          if (!gemm_wait(bar(FULL + st), (it / ST) & 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x73)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a = smem_u32(smem + st * C::STAGE);
          // K-major: 8-row groups 1024 B apart, a K = 16 step is 32 B inside the swizzle atom.
          // MN-major: 64-column blocks 8192 B apart, 8-row groups of k 1024 B, a step is two of them.
          const uint64_t ad = make_sdesc(a, AMN ? 8192 : 16, 1024, SW128);
          const uint64_t bd = make_sdesc(a + C::A_BYTES, BMN ? 8192 : 16, 1024, SW128);
#pragma unroll
          for (int kk = 0; kk < C::BK / 16; ++kk)
            umma_ss_pair(d, ad + (AMN ? 128 : 2) * kk, bd + (BMN ? 128 : 2) * kk, IDESC, (kb - s.k0) | kk);
          umma_commit_pair_mc(bar(EMPTY + st), 0x3);
        }
        if (ok) umma_commit_pair_mc(bar(ACC_FULL + buf), 0x3);
      }
      umma_commit_pair_mc(bar(DRAIN), 0x1);
      gemm_drain(bar(DRAIN), 0, p.wait_limit_ns);
    }
  } else {
    // -------------------------------------------------------------- epilogue (both CTAs)
    const int ew = warp - 2, quarter = warp & 3, chunk = ew >> 2;  // TMEM lane quarter, 64-column chunk
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t acc_empty0 = mapa_shared(bar(ACC_EMPTY), 0);
    uint8_t* stg = smem + C::OFF_STG + ew * C::STG;
    float* bias_s = reinterpret_cast<float*>(smem + C::OFF_BIAS) + ew * 64;
    const long long nb = pack_blocks(p.N);
    uint32_t lt = 0, res_n = 0;
    for (Segments s(p, pair, pairs); s.next(); ++lt) {
      const int buf = lt & 1;
      const int m0 = (s.t / p.tiles_n) * 256 + 128 * static_cast<int>(rank) + quarter * 32;
      const int n = (s.t % p.tiles_n) * BN + chunk * 64;
      const long long row = m0 + lane;
      const bool in_row = row < p.M;
      const bool work = n < p.N && m0 < p.M;  // anything to write (the same for the warp)
      const bool whole = s.whole();
      const bool res_ahead = p.res_tma && work && whole;
      if (p.bias && work && whole) {
        __syncwarp();
        bias_s[lane] = n + lane < p.N ? elem_f32<T>(static_cast<const T*>(p.bias)[n + lane]) : 0.f;
        bias_s[32 + lane] = n + 32 + lane < p.N ? elem_f32<T>(static_cast<const T*>(p.bias)[n + 32 + lane]) : 0.f;
        __syncwarp();
      }
      if (res_ahead && lane == 0) {  // the residual chunk arrives in the staging while the main loop runs
        bulk_wait_read_all();
        fence_proxy_async_smem();  // after the warp's own reads of the staging (a __syncwarp ago)
        mbar_arrive_expect_tx(bar(RES + ew), C::STG);
        tma_load_2d(smem_u32(stg), &p.tma_res, bar(RES + ew), n, m0);
      }
      const bool ok = gemm_wait(bar(ACC_FULL + buf), (lt >> 1) & 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x74);
      bool res_ok = true;
      if (res_ahead) {
        res_ok = gemm_wait(bar(RES + ew), res_n & 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x75);
        if (!res_ok) gemm_drain(bar(RES + ew), res_n & 1, p.wait_limit_ns);
        ++res_n;
      }
      if (!__all_sync(0xffffffffu, ok && res_ok)) break;
      tc_fence_after();
      const uint32_t acc = lane_base + buf * 256u + chunk * 64;
      auto release = [&] {  // this warp's last read of the accumulator is done
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(acc_empty0 + 8u * buf);
      };
      auto load = [&](int h, float (&v)[32]) {
        uint32_t (&raw)[32] = reinterpret_cast<uint32_t (&)[32]>(v);
        tmem_ld32(acc + 32 * h, raw);
        tmem_ld_wait();
      };
      if (!work) {
        release();
        continue;
      }
      const int halves = n + 32 < p.N ? 2 : 1;
      if (!whole) {  // a part of a tile: fp32 sums into the pair's slot
        // (a lane's row is the fastest index but four columns, so that the lanes write neighbouring 16 bytes)
        float4* dst = reinterpret_cast<float4*>(p.partial) +
                      (static_cast<size_t>(2 * pair + (s.k0 ? 0 : 1)) * (BN / 4) + chunk * 16) * 256 + 128 * rank + quarter * 32 + lane;
#pragma unroll 1
        for (int h = 0; h < halves; ++h) {
          float v[32];
          load(h, v);
          if (in_row) {
#pragma unroll
            for (int c = 0; c < 8; ++c)
              dst[(8 * h + c) * 256] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
          }
        }
        release();
        continue;
      }
      if (p.z) {  // the accumulator is read once more below: cheaper than holding it
        staging_free(lane);
#pragma unroll 1
        for (int h = 0; h < halves; ++h) {
          float v[32];
          load(h, v);
          if (p.bias) add_bias(v, bias_s + 32 * h);
          stage32<T>(stg, lane, h, v);
        }
        store_staged(&p.tma_z, p.z_tma, p.z_w, stg, lane, p.z, p.z_stride, m0, n, p.M, p.N);
      }
      if (p.z_codes) {
        // (columns past N hold zeros: W's rows there are read as zeros, the bias too)
        staging_free(lane);
#pragma unroll 1
        for (int h = 0; h < halves; ++h) {
          float v[32];
          load(h, v);
          if (p.bias) add_bias(v, bias_s + 32 * h);
          uint32_t codes[8];
          const uint32_t sc = pack32(v, codes);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint4 w = make_uint4(codes[4 * c], codes[4 * c + 1], codes[4 * c + 2], codes[4 * c + 3]);
            // rows of 64 bytes, 64-byte swizzle
            *reinterpret_cast<uint4*>(stg + lane * 64 + (((2 * h + c) ^ ((lane >> 1) & 3)) << 4)) = w;
          }
          if (in_row) p.z_scales[row * nb + n / 32 + h] = static_cast<uint8_t>(sc);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&p.tma_codes, smem_u32(stg), n, m0);
          bulk_commit_group();
        }
      }
      if (!res_ahead) staging_free(lane);
#pragma unroll 1
      for (int h = 0; h < halves; ++h) {
        float v[32];
        load(h, v);
        if (h == halves - 1) release();
        if (p.bias) add_bias(v, bias_s + 32 * h);
        act_any(p.act, v);
        if (res_ahead) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float f[8];
            unpack8<T>(*stage_part(stg, lane, 4 * h + c), f);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[8 * c + e] += f[e];
          }
        } else if (p.res && in_row) {
          const T* rp = static_cast<const T*>(p.res) + row * p.res_stride + n + 32 * h;
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (n + 32 * h + i < p.N) v[i] += elem_f32<T>(rp[i]);
        }
        stage32<T>(stg, lane, h, v);
      }
      store_staged(&p.tma_out, p.out_tma, p.out_w, stg, lane, p.out, p.out_stride, m0, n, p.M, p.N);
    }
    if (lane == 0) bulk_wait_all();  // output written before the CTA ends
  }
  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while its pair may still signal it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Joins the parts of split tiles in the order of k and applies the epilogue: 32 columns
// of a row per thread, the rows of a warp's threads neighbours.
template <int BN, typename T>
__global__ void __launch_bounds__(256) gemm_finish_kernel(const __grid_constant__ GemmParams p) {
  const int t = blockIdx.x;
  const int first = static_cast<int>(static_cast<long long>(t) * p.nk / p.split);
  const int last = static_cast<int>((static_cast<long long>(t + 1) * p.nk - 1) / p.split);
  if (first == last) {  // one pair computed the whole tile
    griddep_wait();
    return;
  }
  __shared__ __align__(16) uint8_t stage[8][2048];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.y * 8 + warp;  // of 32 rows x 32 columns
  const int r = unit % 8 * 32 + lane, c = unit / 8 * 32;
  const long long m = static_cast<long long>(t / p.tiles_n) * 256 + unit % 8 * 32;
  const int n = (t % p.tiles_n) * BN + c;
  griddep_wait();
  griddep_launch_dependents();
  if (m >= p.M || n >= p.N) return;
  float v[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = 0.f;
  if (m + lane < p.M) {
    for (int q = first; q <= last; ++q) {
      const long long b = static_cast<long long>(q) * p.split;
      const int slot = 2 * q + (b > static_cast<long long>(t) * p.nk ? 0 : 1);  // began inside the tile, or before or at its first step
      const float4* src = reinterpret_cast<const float4*>(p.partial) + (static_cast<size_t>(slot) * (BN / 4) + c / 4) * 256 + r;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 x = __ldcg(src + i * 256);
        v[4 * i] += x.x;
        v[4 * i + 1] += x.y;
        v[4 * i + 2] += x.z;
        v[4 * i + 3] += x.w;
      }
    }
  }
  __syncwarp();
  finish_piece<T>(p, m, n, lane, stage[warp], v);
}

// ------------------------------------------------------------------ small products
// One CTA per 128 x 64 tile of D, and per cluster of S CTAs one tile: each of the S takes
// a share of the reduction, so that a product of few rows (a single token reads W and
// little else) or a short one still has every SM loading, with all of a CTA's steps on
// their way at once. The S sums meet through distributed shared memory, in the order
// of the ranks, and each CTA finishes a part of the tile. No second kernel, no sums in
// global memory.
struct SmallCfg {
  static constexpr int BM = 128, BN = 64, BK = 64;
  static constexpr int A_BYTES = BM * BK * 2, B_BYTES = BN * BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int ST = 4;
  static constexpr int SUM_BYTES = BM * BN * 4;  // this CTA's sums, over the first stages' place
  static constexpr int OFF_BAR = ST * STAGE;
  static constexpr int SMEM = OFF_BAR + 128 + 1024;
  static constexpr int THREADS = 192;  // warp 0 TMA, warp 1 MMA, warps 2-5 epilogue
  static_assert(SUM_BYTES + 4 * 2048 <= ST * STAGE, "sums and the warps' staging fit");
};

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}

template <bool AMN, bool BMN, typename T>
__global__ void __launch_bounds__(SmallCfg::THREADS) gemm_small_kernel(const __grid_constant__ GemmParams p) {
  using C = SmallCfg;
  constexpr int ST = C::ST;
  constexpr bool kBF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC = make_idesc_f16(kBF16, C::BM, C::BN, BMN) | (AMN ? 1u << 15 : 0u);
  constexpr uint32_t SW128 = 2;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  auto bar = [&](int i) { return smem_u32(bars + i); };
  const int FULL = 0, EMPTY = ST, ACC = 2 * ST;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * ST + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.split, rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int tile = static_cast<int>(blockIdx.x) / S;
  const int m0 = (tile / p.tiles_n) * C::BM, n0 = (tile % p.tiles_n) * C::BN;
  const int k0 = static_cast<int>(static_cast<long long>(p.nk) * rank / S), k1 = static_cast<int>(static_cast<long long>(p.nk) * (rank + 1) / S);
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST; ++i) {
      mbar_init(bar(FULL + i), 1);
      mbar_init(bar(EMPTY + i), 1);
    }
    mbar_init(bar(ACC), 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tma_a);
    tma_prefetch_desc(&p.tma_b);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), 64);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();
  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int st = it % ST;
        if (!gemm_wait(bar(EMPTY + st), ((it / ST) & 1) ^ 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x76)) break;
        const uint32_t a = smem_u32(smem + st * C::STAGE), b = a + C::A_BYTES;
        mbar_arrive_expect_tx(bar(FULL + st), p.a_bytes + C::B_BYTES);
        if constexpr (AMN) {
          tma_load_2d(a, &p.tma_a, bar(FULL + st), m0, kb * C::BK);
          tma_load_2d(a + 8192, &p.tma_a, bar(FULL + st), m0 + 64, kb * C::BK);
        } else {  // (boxes of as many rows as M has; the rest of the tile's rows go nowhere)
          tma_load_2d(a, &p.tma_a, bar(FULL + st), kb * C::BK, m0);
        }
        if constexpr (BMN) tma_load_2d(b, &p.tma_b, bar(FULL + st), n0, kb * C::BK);
        else tma_load_2d(b, &p.tma_b, bar(FULL + st), kb * C::BK, n0);
      }
      for (int i = it > ST ? it - ST : 0; i < it; ++i) gemm_drain(bar(FULL + i % ST), (i / ST) & 1, p.wait_limit_ns);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      int it = 0;
      for (int kb = k0; kb < k1; ++kb, ++it) {
        const int st = it % ST;
        if (!gemm_wait(bar(FULL + st), (it / ST) & 1, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x77)) break;
        tc_fence_after();
        const uint32_t a = smem_u32(smem + st * C::STAGE);
        const uint64_t ad = make_sdesc(a, AMN ? 8192 : 16, 1024, SW128);
        const uint64_t bd = make_sdesc(a + C::A_BYTES, BMN ? 8192 : 16, 1024, SW128);
#pragma unroll
        for (int kk = 0; kk < C::BK / 16; ++kk)
          umma_ss(tmem, ad + (AMN ? 128 : 2) * kk, bd + (BMN ? 128 : 2) * kk, IDESC, it | kk);
        umma_commit(bar(EMPTY + st));
      }
      umma_commit(bar(ACC));  // (after a timeout too: it then only says that the MMAs issued are done)
      gemm_drain(bar(ACC), 0, p.wait_limit_ns);
    }
  }
  __syncwarp();
  const int quarter = warp & 3;
  const bool rows = warp >= 2 && m0 + quarter * 32 < p.M;  // an epilogue warp with rows of D
  bool ok = true;
  if (rows) {
    ok = __all_sync(0xffffffffu, gemm_wait(bar(ACC), 0, p, abort_flag, FRATTN_STATUS_WAIT_TIMEOUT | 0x78));
    tc_fence_after();
  }
  const uint32_t acc = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  uint8_t* stg = smem + C::SUM_BYTES + quarter * 2048;  // (free once all MMAs are done)
  if (S == 1) {
    if (rows && ok) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        if (n0 + 32 * h >= p.N) break;
        float v[32];
        tmem_ld32(acc + 32 * h, reinterpret_cast<uint32_t (&)[32]>(v));
        tmem_ld_wait();
        finish_piece<T>(p, m0 + quarter * 32, n0 + 32 * h, lane, stg, v);
      }
    }
  } else {
    // (the stages' place: all MMAs, the stages' readers, are done when ACC has completed)
    float4* sums = reinterpret_cast<float4*>(smem);  // [16 groups of 4 columns][128 rows]
    if (rows && ok) {
#pragma unroll 1
      for (int h = 0; h < 2; ++h) {
        float v[32];
        tmem_ld32(acc + 32 * h, reinterpret_cast<uint32_t (&)[32]>(v));
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < 8; ++c)
          sums[(8 * h + c) * 128 + quarter * 32 + lane] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
      }
    }
    cluster_sync_all();  // every CTA's sums are written (a CTA without rows or timed out has none to read)
    // this CTA's share of the tile's (row, 32 columns) units
    if (warp >= 2) {
      const int share = 256 / S;  // 32 rows a warp at a time: a multiple of 32
      for (int u = rank * share + (warp - 2) * 32; u < (rank + 1) * share; u += 128) {
        const int r = u & 127, h = u >> 7, n = n0 + 32 * h;
        if (m0 + r >= p.M || n >= p.N) continue;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
        if (m0 + r + lane < p.M) {
          for (int q = 0; q < S; ++q) {
            const uint32_t from = mapa_shared(smem_u32(sums + (8 * h) * 128 + r + lane), q);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
              const float4 x = ld_cluster_f4(from + c * 128 * 16);
              v[4 * c] += x.x;
              v[4 * c + 1] += x.y;
              v[4 * c + 2] += x.z;
              v[4 * c + 3] += x.w;
            }
          }
        }
        __syncwarp();
        finish_piece<T>(p, m0 + r, n, lane, stg, v);
      }
    }
    cluster_sync_all();  // nobody leaves while its sums may be read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 64);
  }
}

// ---------------------------------------------------------------- host
// One operand or output of a product: rows of `stride` elements.
struct Mat {
  const void* p;
  long long stride;
};

int encode_map(CUtensorMap* m, const void* base, long long cols, long long rows, long long stride, int box_cols,
               int box_rows, bool bf16) {
  const TmapEncodeFn enc = tmap_encoder();
  if (!enc) return FRATTN_E_TMAP;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : FRATTN_E_TMAP;
}

// Codes of a checkpoint: rows of 32 nb bytes.
int encode_codes_map(CUtensorMap* m, const void* base, long long cols, long long rows) {
  const TmapEncodeFn enc = tmap_encoder();
  if (!enc) return FRATTN_E_TMAP;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols)};
  cuuint32_t box[2] = {64, 32};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : FRATTN_E_TMAP;
}

bool rows16(const void* p, long long stride) { return aligned_to(p, 16) && stride % 8 == 0; }

int sm_pairs() {
  const int n = sm_count_for_current_device();
  return (n > 1 ? n : 148) / 2;
}

// Tile width and split of an M x N product over nk steps of 64.
struct GemmPlan {
  int bn, tiles, split, pairs;  // bn 64: the small kernel, split its CTAs per tile
  size_t partial_bytes;
};

// The shortest of four estimates, in microseconds of a 64-wide step: whole tiles, dealt
// out in rounds of all pairs, and the same steps dealt out evenly (Segments), for tiles
// 256 and 128 wide. With every pair at work a step is bound by what the SMs draw from
// L2: 0.37 us for 256 x 256 (64 KB) but 0.31 for 256 x 128 (48 KB), measured at
// 9216 x 3424 -> 1280 (71 us with 256-wide tiles in three rounds, 90 us with 128-wide
// ones in five); narrow tiles pay only where there are too few wide ones. Even dealing
// pays for writing and reading the parts (4 TB/s together) and a second kernel.
GemmPlan gemm_plan(int M, int N, int nk) {
  GemmPlan best{};
  const int P = sm_pairs();
  double best_us = 1e30;
  {
    // 128 x 64 tiles, up to 8 CTAs on one while that leaves each two steps, and all of them
    // run at once: two fit an SM, but clusters of 8 have to fit its processing cluster
    // too, so that 37 clusters of 8 took two rounds (21 us; 10 with 4). Bound by 24 KB
    // from L2 a step (10 TB/s for all), or by latency.
    const long long tiles = static_cast<long long>((M + 127) / 128) * ((N + 63) / 64);
    int S = 1;
    while (S < 8 && tiles * 2 * S <= 3 * P && nk >= 4 * S) S *= 2;
    const double rows = M < 128 ? M : 128;
    const double us = tiles * nk * (rows * 128 + 8192) / 10e6 + 0.25 * ((nk + S - 1) / S) * ((tiles * S + 4 * P - 1) / (4 * P)) + 1.0;
    if (tiles * S < (1 << 30)) {
      best_us = us;
      best = GemmPlan{64, static_cast<int>(tiles), S, 0, 0};
    }
  }
  for (int bn : {256, 128}) {
    const long long tiles = static_cast<long long>((M + 255) / 256) * ((N + bn - 1) / bn);
    if (tiles > (1 << 30) / (nk + 1)) continue;
    const double step_us = bn == 256 ? 0.37 : 0.31;
    {
      const long long rounds = (tiles + P - 1) / P;
      const double us = static_cast<double>(rounds) * nk * step_us + 4.0;  // (filling, the last tile's epilogue)
      if (us < best_us) {
        best_us = us;
        best = GemmPlan{bn, static_cast<int>(tiles), 0, static_cast<int>(tiles < P ? tiles : P), 0};
      }
    }
    const long long total = tiles * nk;
    int split = static_cast<int>((total + P - 1) / P);
    if (split < 4) split = 4;
    if (tiles % P != 0) {
      const int pairs = static_cast<int>((total + split - 1) / split);
      const double rows = M < 256 ? M : 256;
      const double us = split * step_us + 8.0 + 2.0 * pairs * rows * bn * 4 * 2 / 4e6;
      if (us < best_us) {
        best_us = us;
        best = GemmPlan{bn, static_cast<int>(tiles), split, pairs, static_cast<size_t>(2) * pairs * 256 * bn * 4};
      }
    }
  }
  return best;
}

template <int BN, bool AMN, bool BMN, typename T>
int gemm_launch(GemmParams& p, const GemmPlan& plan, cudaStream_t st) {
  using C = GemmCfg<BN>;
  auto kern = gemm_pair_kernel<BN, AMN, BMN, T>;
  static unsigned long long attr_set = 0;  // per device; setting twice is harmless
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bitv = 1ull << (dev & 63);
  if (!(attr_set & bitv)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess)
      return FRATTN_E_CUDA;
    attr_set |= bitv;
  }
  const int rc = launch_overlapped(kern, dim3(2 * plan.pairs), dim3(C::THREADS), C::SMEM, st, 2, p);
  if (rc || !plan.split) return rc;
  return launch_overlapped(gemm_finish_kernel<BN, T>, dim3(plan.tiles, BN / 32), dim3(256), 0, st, 1, p);
}

template <bool AMN, bool BMN, typename T>
int gemm_small_launch(const GemmParams& p, const GemmPlan& plan, cudaStream_t st) {
  auto kern = gemm_small_kernel<AMN, BMN, T>;
  static unsigned long long attr_set = 0;
  int dev = 0;
  cudaGetDevice(&dev);
  const unsigned long long bitv = 1ull << (dev & 63);
  if (!(attr_set & bitv)) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SmallCfg::SMEM) != cudaSuccess)
      return FRATTN_E_CUDA;
    attr_set |= bitv;
  }
  return launch_overlapped(kern, dim3(plan.tiles * plan.split), dim3(SmallCfg::THREADS), SmallCfg::SMEM, st, plan.split, p);
}

// D[M, N] = A B^T with the epilogue in p (bias .. z_scales set by the caller). A is
// [M, K] rows (or [K, M] with AMN), B [N, K] (or [K, N] with BMN), 16-byte rows.
template <bool AMN, bool BMN, typename T>
int gemm(GemmParams& p, const Mat& a, const Mat& b, int M, int N, int K, void* ws, size_t ws_bytes, int32_t* status,
         cudaStream_t st) {
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  p.M = M;
  p.N = N;
  p.nk = (K + 63) / 64;
  const GemmPlan plan = gemm_plan(M, N, p.nk);
  if (!plan.bn) return FRATTN_E_SHAPE;
  if (plan.partial_bytes > ws_bytes) return FRATTN_E_WORKSPACE;
  p.tiles_n = (N + plan.bn - 1) / plan.bn;
  p.tiles = plan.tiles;
  p.split = plan.split;
  p.partial = static_cast<float*>(ws);
  p.status = status;
  p.wait_limit_ns = frattn_wait_limit_ns();
  const bool small = plan.bn == 64;
  const int a_rows = small && M < 128 ? (M + 7) / 8 * 8 : 128;  // of a K-major A in a box
  p.a_bytes = AMN ? SmallCfg::A_BYTES : a_rows * 128;
  if (encode_map(&p.tma_a, a.p, AMN ? M : K, AMN ? K : M, a.stride, 64, AMN ? 64 : a_rows, bf16) ||
      encode_map(&p.tma_b, b.p, BMN ? N : K, BMN ? K : N, b.stride, 64, BMN || small ? 64 : plan.bn / 2, bf16))
    return FRATTN_E_TMAP;
  auto width = [&](const void* q, long long stride) {
    for (int w = 8; w > 1; w >>= 1)
      if (aligned_to(q, 2 * w) && stride % w == 0 && N % w == 0) return w;
    return 1;
  };
  p.out_tma = rows16(p.out, p.out_stride);
  p.out_w = width(p.out, p.out_stride);
  if (p.out_tma && !small && encode_map(&p.tma_out, p.out, N, M, p.out_stride, 64, 32, bf16)) return FRATTN_E_TMAP;
  if (p.z) {
    p.z_tma = rows16(p.z, p.z_stride);
    p.z_w = width(p.z, p.z_stride);
    if (p.z_tma && !small && encode_map(&p.tma_z, p.z, N, M, p.z_stride, 64, 32, bf16)) return FRATTN_E_TMAP;
  }
  if (p.z_codes && !small && encode_codes_map(&p.tma_codes, p.z_codes, pack_blocks(N) * kPackBlock, M)) return FRATTN_E_TMAP;
  p.res_vec = p.res && rows16(p.res, p.res_stride);
  if (small) return gemm_small_launch<AMN, BMN, T>(p, plan, st);
  p.res_tma = p.res && rows16(p.res, p.res_stride) && p.res_stride >= N && !p.z && !p.z_codes;
  if (p.res_tma && encode_map(&p.tma_res, p.res, N, M, p.res_stride, 64, 32, bf16)) return FRATTN_E_TMAP;
  if (plan.bn == 256) return gemm_launch<256, AMN, BMN, T>(p, plan, st);
  return gemm_launch<128, AMN, BMN, T>(p, plan, st);
}

size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

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
// blockIdx.y + gridDim.y, ...): neighbouring threads read neighbouring vectors, the
// column sums stay in registers, and the next R rows are on their way while R rows are
// worked on.
template <typename T, int VEC, int ACT, bool PACKED>
__global__ void __launch_bounds__(256, 2) act_bwd_kernel(const ActBwdParams p) {
  constexpr int R = 4;
  const int v = blockIdx.x * blockDim.x + threadIdx.x;
  griddep_wait();
  griddep_launch_dependents();
  if (v * VEC >= p.N) return;
  const size_t c = static_cast<size_t>(v) * VEC;
  const int nb = static_cast<int>(pack_blocks(p.N));
  float sum[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) sum[e] = 0.f;
  const long long step = gridDim.y;
  Vec<T, VEC> ndy[R], nz[R];
  CodeVec<VEC> nq[R];
  uint32_t nscale[R];
  auto fetch = [&](long long row0) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row < p.T) {
        ndy[r].load(static_cast<const T*>(p.dout) + row * p.dout_stride + c);
        if constexpr (ACT != FRATTN_ACT_NONE) {
          if constexpr (PACKED) {
            nq[r].load(p.z_codes + row * nb * kPackBlock + c);
            nscale[r] = __ldcg(p.z_scales + row * nb + v * VEC / kPackBlock);
          } else {
            nz[r].load(static_cast<const T*>(p.z) + row * p.z_stride + c);
          }
        }
      }
    }
  };
  fetch(blockIdx.y);
  for (long long row0 = blockIdx.y; row0 < p.T; row0 += step * R) {
    Vec<T, VEC> dy[R], z[R];
    CodeVec<VEC> q[R];
    uint32_t scale[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      dy[r] = ndy[r];
      if constexpr (ACT != FRATTN_ACT_NONE) {
        if constexpr (PACKED) {
          q[r] = nq[r];
          scale[r] = nscale[r];
        } else {
          z[r] = nz[r];
        }
      }
    }
    fetch(row0 + step * R);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const long long row = row0 + r * step;
      if (row >= p.T) break;
      float d[VEC];
      dy[r].get(d);
      if constexpr (ACT != FRATTN_ACT_NONE) {
        float f[VEC];
        if constexpr (PACKED) q[r].get(pack_step(scale[r]), f);
        else z[r].get(f);
#pragma unroll
        for (int e = 0; e + 1 < VEC; e += 2) act_grad_f2<ACT>(f[e], f[e + 1], d[e], d[e + 1]);
        if constexpr (VEC == 1) {
          float none = 0.f;
          act_grad_f2<ACT>(f[0], 0.f, d[0], none);
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sum[e] += d[e];
      if (p.dz) Vec<T, VEC>::put(static_cast<T*>(p.dz) + row * p.dz_stride + c, d);
    }
  }
  if (p.partial) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) p.partial[static_cast<size_t>(blockIdx.y) * p.N + c + e] = sum[e];
  }
}

// Strips of rows, and partial rows of the bias gradient: two blocks of 256 threads to an
// SM with four rows each on their way are enough for the memory, and more strips cost
// more partial sums (592 of them took 8 us to add up at N = 3424).
constexpr int kMaxStrips = 296;

template <typename T, int VEC, int ACT, bool PACKED>
int act_bwd_launch(const ActBwdParams& p, int* groups, cudaStream_t st) {
  const int nv = p.N / VEC;
  const int tiles = (nv + 255) / 256;
  const int bx = ((nv + tiles - 1) / tiles + 31) / 32 * 32;
  const int gx = (nv + bx - 1) / bx;
  long long gy = static_cast<long long>(sm_count_for_current_device()) * (512 / bx) / gx;
  const long long rows4 = (p.T + 3) / 4;
  if (gy > rows4) gy = rows4;
  if (gy > kMaxStrips) gy = kMaxStrips;
  if (gy < 1) gy = 1;
  *groups = static_cast<int>(gy);
  return launch_overlapped(act_bwd_kernel<T, VEC, ACT, PACKED>, dim3(gx, static_cast<unsigned>(gy)), dim3(bx), 0, st, 1, p);
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
  if (rv.v == 2) return p.z_codes ? act_bwd_act<T, 2, true>(p, act, groups, st) : act_bwd_act<T, 2, false>(p, act, groups, st);
  return p.z_codes ? act_bwd_act<T, 1, true>(p, act, groups, st) : act_bwd_act<T, 1, false>(p, act, groups, st);
}

// Workspace of the backward pass: dz [T, Np] (rows padded to 16 bytes), partial
// column sums, the 16-bit values of a packed x [T, Kp], and the parts of split tiles
// (of one product at a time).
struct BwdLayout {
  long long np, kp;
  size_t dz, partial, x, gemm, gemm_bytes, total;
};
BwdLayout bwd_layout(int T, int K, int N) {
  BwdLayout l;
  l.np = (static_cast<long long>(N) + 7) / 8 * 8;
  l.kp = (static_cast<long long>(K) + 7) / 8 * 8;
  l.dz = 0;
  l.partial = up256(static_cast<size_t>(T) * l.np * 2);
  l.x = l.partial + up256(static_cast<size_t>(kMaxStrips) * N * sizeof(float));
  l.gemm = l.x + up256(static_cast<size_t>(T) * l.kp * 2);
  const size_t dx = gemm_plan(T > 0 ? T : 1, K, (N + 63) / 64).partial_bytes;
  const size_t dw = gemm_plan(N, K, T > 0 ? (T + 63) / 64 : 1).partial_bytes;
  l.gemm_bytes = dx > dw ? dx : dw;
  l.total = l.gemm + up256(l.gemm_bytes);
  return l;
}

template <typename T>
int linear_bwd(const void* dout, long long dout_stride, const void* x, long long x_stride, const int8_t* x_codes,
               const uint8_t* x_scales, const void* w, long long w_stride, const void* z, long long z_stride,
               const int8_t* z_codes, const uint8_t* z_scales, int act, int rows, int K, int N, int dtype, void* dx,
               long long dx_stride, void* dw, void* db, uint8_t* ws, int32_t* status, cudaStream_t st) {
  const BwdLayout l = bwd_layout(rows, K, N);
  const bool in_place = act == FRATTN_ACT_NONE && rows16(dout, dout_stride) && dout_stride >= N;
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
  GemmParams m;
  if (dx && rows > 0) {
    memset(&m, 0, sizeof(m));
    m.out = dx;
    m.out_stride = dx_stride;
    const Mat a{dz, dz_stride}, b{w, w_stride};
    if ((rc = gemm<false, true, T>(m, a, b, rows, K, N, ws + l.gemm, l.gemm_bytes, status, st))) return rc;
  }
  if (dw) {
    if (rows == 0) return cudaMemsetAsync(dw, 0, static_cast<size_t>(N) * K * 2, st) == cudaSuccess ? 0 : FRATTN_E_CUDA;
    if (x_codes) {
      if ((rc = act_unpack(x_codes, x_scales, rows, K, dtype, ws + l.x, l.kp, st))) return rc;
      x = ws + l.x;
      x_stride = l.kp;
    }
    memset(&m, 0, sizeof(m));
    m.out = dw;
    m.out_stride = K;
    const Mat a{dz, dz_stride}, b{x, x_stride};
    return gemm<true, true, T>(m, a, b, N, K, rows, ws + l.gemm, l.gemm_bytes, status, st);
  }
  return 0;
}

}  // namespace
}  // namespace frattn

using namespace frattn;

extern "C" {

int frattn_workspace_bytes_linear_act(int T, int K, int N, size_t* bytes) {
  if (!bytes) return FRATTN_E_NULL;
  if (T < 0 || K <= 0 || N <= 0) return FRATTN_E_SHAPE;
  *bytes = T > 0 ? gemm_plan(T, N, (K + 63) / 64).partial_bytes : 0;
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
  if (need && !workspace) return FRATTN_E_NULL;
  if (!aligned_to(workspace, 256)) return FRATTN_E_ALIGN;
  GemmParams m;
  memset(&m, 0, sizeof(m));
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
  const Mat a{x, x_stride}, b{w, w_stride};
  if (dtype == FRATTN_BF16)
    return gemm<false, false, __nv_bfloat16>(m, a, b, T, N, K, workspace, workspace_bytes, status, st);
  return gemm<false, false, __half>(m, a, b, T, N, K, workspace, workspace_bytes, status, st);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (dtype == FRATTN_BF16)
    return linear_bwd<__nv_bfloat16>(dout, dout_stride, x, x_stride, x_codes, x_scales, w, w_stride, z, z_stride,
                                     z_codes, z_scales, activation, T, K, N, dtype, dx, dx_stride, dw, db, ws, status, st);
  return linear_bwd<__half>(dout, dout_stride, x, x_stride, x_codes, x_scales, w, w_stride, z, z_stride, z_codes,
                            z_scales, activation, T, K, N, dtype, dx, dx_stride, dw, db, ws, status, st);
}

}  // extern "C"
