// Product of 8-bit integer rows with scales for each token and each channel.
//
//   out[m, n] = sa[m] * sb[n] * sum_k a[m, k] * b[n, k]  (+ bias[n])
//
// a [M, K] and b [N, K] are int8 with K contiguous. The sum is exact in int32
// (|sum| <= 2^14 K < 2^31 for K < 2^17), the scales and the bias are applied
// in fp32 and the result is rounded once to the output's type.
#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxK = (1 << 17) - 1;
constexpr int64_t kMaxRows = (int64_t(1) << 31) - 512;  // a tile's last row stays in 32 bits

struct I8Args {
  const int8_t* a;
  const int8_t* b;
  const float* sa;
  const float* sb;
  const void* bias;
  void* out;
  int64_t lda, ldb, ldo;
  int32_t m, n, k, out_type, bias_type;
};

// 16 bytes of a row from byte k on, from any address (gfx950 loads 16 bytes
// at any alignment); bytes at or past K read as zero and are not touched.
__device__ __forceinline__ i32x4 load16(const int8_t* row, int k, int K) {
  i32x4 v = {0, 0, 0, 0};
  const int n = K - k;
  if (n >= 16) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (n > 0) {
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 15; ++i)
      if (i < n) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
    v = i32x4{static_cast<int>(w[0]), static_cast<int>(w[1]), static_cast<int>(w[2]), static_cast<int>(w[3])};
  }
  return v;
}

__device__ __forceinline__ float load_any(const void* p, int type, int64_t at) {
  if (type == MM_T_FP32) return static_cast<const float*>(p)[at];
  if (type == MM_T_FP16) return static_cast<float>(static_cast<const _Float16*>(p)[at]);
  return static_cast<float>(static_cast<const bf16*>(p)[at]);
}

__device__ __forceinline__ void store_any(void* p, int type, int64_t at, float v) {
  if (type == MM_T_FP32)
    static_cast<float*>(p)[at] = v;
  else if (type == MM_T_FP16)
    static_cast<_Float16*>(p)[at] = static_cast<_Float16>(v);
  else
    static_cast<bf16*>(p)[at] = static_cast<bf16>(v);
}

// LDS tile [ROWS][128 bytes]: 16-byte slot s of row r sits at s ^ ((r >> 1) & 7),
// which gives the 16 rows of one pass of a fragment read distinct banks.
constexpr int BK = 128;
__device__ __forceinline__ int slot_of(int r, int s) { return r * BK + ((s ^ ((r >> 1) & 7)) << 4); }

// 128 x 128 tile, 4 waves of 64 x 64 in v_mfma_i32_32x32x32_i8 blocks. The
// operands are swapped, so a lane holds 4 consecutive columns of one row.
__global__ __launch_bounds__(256) void int8_tile_kernel(I8Args p) {
  constexpr int BM = 128, BN = 128;
  __shared__ __attribute__((aligned(16))) int8_t As[BM * BK], Bs[BN * BK];
  const int num_n = (p.n + BN - 1) / BN;
  const int m0 = blockIdx.x / num_n * BM, n0 = blockIdx.x % num_n * BN;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int8_t *pa[4], *pb[4];
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const int r = (v * 256 + tid) >> 3;
    pa[v] = p.a + static_cast<int64_t>(min(m0 + r, p.m - 1)) * p.lda;
    pb[v] = p.b + static_cast<int64_t>(min(n0 + r, p.n - 1)) * p.ldb;
  }
  const int s = tid & 7;
  i32x4 ra[4], rb[4];
  auto load = [&](int k0) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      ra[v] = load16(pa[v], k0 + s * 16, p.k);
      rb[v] = load16(pb[v], k0 + s * 16, p.k);
    }
  };
  i32x16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;
  load(0);
  for (int k0 = 0; k0 < p.k; k0 += BK) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = (v * 256 + tid) >> 3;
      *reinterpret_cast<i32x4*>(As + slot_of(r, s)) = ra[v];
      *reinterpret_cast<i32x4*>(Bs + slot_of(r, s)) = rb[v];
    }
    __syncthreads();
    if (k0 + BK < p.k) load(k0 + BK);
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      i32x4 fa[2], fb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[i] = *reinterpret_cast<const i32x4*>(As + slot_of(wm * 64 + i * 32 + (lane & 31), kk * 2 + (lane >> 5)));
        fb[i] = *reinterpret_cast<const i32x4*>(Bs + slot_of(wn * 64 + i * 32 + (lane & 31), kk * 2 + (lane >> 5)));
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[j], fa[i], acc[i][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = m0 + wm * 64 + i * 32 + (lane & 31);
    if (row >= p.m) continue;
    const float sa = p.sa[row];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int col = n0 + wn * 64 + j * 32 + (r >> 2) * 8 + (lane >> 5) * 4 + (r & 3);
        if (col >= p.n) continue;
        float v = static_cast<float>(acc[i][j][r]) * sa * p.sb[col];
        if (p.bias) v += load_any(p.bias, p.bias_type, col);
        store_any(p.out, p.out_type, static_cast<int64_t>(row) * p.ldo + col, v);
      }
  }
}

bool is_float_type(int t) { return t == MM_T_BF16 || t == MM_T_FP16 || t == MM_T_FP32; }

}  // namespace

extern "C" int mm_int8_matmul(const int8_t* a, int64_t lda, const int8_t* b, int64_t ldb, const float* a_scale,
                              const float* b_scale, const void* bias, int32_t bias_type, int64_t m, int64_t n,
                              int64_t k, void* out, int64_t ldo, int32_t out_type, mm_stream_t stream) {
  MM_CHECK_ARG(m >= 0 && n > 0 && k > 0 && k <= kMaxK && m < kMaxRows && n < kMaxRows,
               "mm_int8_matmul: bad sizes (%lld x %lld x %lld; K at most %d)", static_cast<long long>(m),
               static_cast<long long>(n), static_cast<long long>(k), kMaxK);
  MM_CHECK_ARG(is_float_type(out_type) && (!bias || is_float_type(bias_type)), "mm_int8_matmul: bad types");
  MM_CHECK_ARG((m <= 1 || lda >= k) && (n <= 1 || ldb >= k) && (m <= 1 || ldo >= n), "mm_int8_matmul: bad strides");
  const int64_t tiles = ((m + 127) / 128) * ((n + 127) / 128);
  MM_CHECK_ARG(tiles < (int64_t(1) << 24), "mm_int8_matmul: too many tiles");  // 2^32 threads in a launch
  if (m == 0) return MM_OK;
  MM_CHECK_ARG(a && b && a_scale && b_scale && out, "mm_int8_matmul: null pointer");
  const I8Args p{a, b, a_scale, b_scale, bias, out, lda, ldb, ldo, static_cast<int32_t>(m), static_cast<int32_t>(n),
                 static_cast<int32_t>(k), out_type, bias_type};
  int8_tile_kernel<<<static_cast<uint32_t>(tiles), 256, 0, mm_hip_stream(stream)>>>(p);
  return mm_check_launch("int8_tile_kernel");
}
