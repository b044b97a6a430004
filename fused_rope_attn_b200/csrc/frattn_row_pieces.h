// A row of any alignment as the 16-byte pieces of memory that it touches. Plain C++: the
// kernels and the host's test of the arithmetic share it.
#pragma once

#if defined(__CUDACC__)
#define FRATTN_HD __host__ __device__ __forceinline__
#else
#define FRATTN_HD inline
#endif

namespace frattn {

// The row's `bytes` bytes start `off` (< 16) bytes into their first piece. Thread t of n calls
// copy(at, from, size) for its pieces: 16 bytes go to `at`, `size` of them from `from` and
// zeros for the rest; both are counted from the first piece and multiples of 16. The
// pieces end with one of zeros (size 0), which gives the first piece as its source: an
// asynchronous copy wants an aligned address even where it reads nothing.
template <typename F>
FRATTN_HD void row_pieces(int off, int bytes, int t, int n, F&& copy) {
  const int end = off + bytes;
  for (int at = 16 * t; at < end + 16; at += 16 * n) {
    const int left = end - at;
    copy(at, left > 0 ? at : 0, left < 16 ? (left > 0 ? left : 0) : 16);
  }
}

}  // namespace frattn
