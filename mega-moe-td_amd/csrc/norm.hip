// Root-mean-square norm of rows with the residual's addition, its backward,
// and rows in 8 bits with one scale each.
//
//   h = round(x + residual)          (h = x without a residual)
//   y = h * r * w,  r = 1 / sqrt(mean(h^2) + eps)
//   8 bits: s = max(a, 1e-30) / Q with a = max |y| over the row (s = 1 where
//           a = 0), q = round(y / s); Q = 127 (int8) or 448 (E4M3)
//   backward: dx = dh + r w dy - h r^3 mean(w dy h),  dw = sum_rows dy h r
//
// The norm is taken of h as it is stored, so that the backward (which reads h)
// and a caller who adds and norms in two steps compute the same function. Sums
// and statistics are fp32; each output is rounded once.
//
// Memory bound: every element is read once and written once. A row stays in
// the registers of its TPR threads (NV vectors of 8 columns each) between the
// sum of squares, the maximum and the output.
#include "common.h"

namespace {

struct NormArgs {
  const void* x;
  const void* res;     // or NULL
  const void* w;       // or NULL
  void* h;             // stored sum, given with res
  void* y;
  float* scale;        // per row, 8-bit outputs
  float* rstd;         // per row, or NULL
  int64_t ldx, ldr, rows;
  int32_t hidden, w_type, y_type, norm;
  float eps;
};

struct NormBwdArgs {
  const void* dy;
  const void* dh;      // or NULL
  const void* h;
  const void* w;       // or NULL
  const float* rstd;
  void* dx;
  void* dres;          // dx in the residual's type, or NULL
  float* partial;      // [gridDim.x, hidden], or NULL
  int64_t lddy, lddh, ldh, rows;
  int32_t hidden, w_type;
};

constexpr float kScaleFloor = 1e-30f;  // below it a row's scale would leave the normal range

// Eight consecutive elements from any address the type's own alignment allows
// (one or two 16-byte loads), the last vector of a row element by element.
template <class T>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, float* f) {
  if (n >= 8) {
    T v[8];
    __builtin_memcpy(v, p, sizeof(v));
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
  }
}

template <class T>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const T* v) {
  if (n >= 8) {
    __builtin_memcpy(p, v, 8 * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = v[i];
  }
}

template <class T>
__device__ __forceinline__ void store8_f32(T* __restrict__ p, int n, const float* f) {
  T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(f[i]);
  store8(p, n, v);
}

__device__ __forceinline__ void load8_any(const void* p, int type, int64_t at, int n, float* f) {
  if (type == MM_T_FP32)
    load8(static_cast<const float*>(p) + at, n, f);
  else if (type == MM_T_FP16)
    load8(static_cast<const _Float16*>(p) + at, n, f);
  else
    load8(static_cast<const bf16*>(p) + at, n, f);
}

// Reductions over the TPR threads of a row; every thread gets the result.
// `lds` has one slot per wave; calls alternate between two such arrays, so a
// slot is rewritten only after a later call's barrier.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += lds[i];
  }
  return v;
}

template <int TPR>
__device__ __forceinline__ uint32_t row_umax(uint32_t v, uint32_t* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m)));
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v = max(v, lds[i]);
  }
  return v;
}

template <int TPR>
constexpr int norm_threads() { return TPR < 256 ? 256 : TPR; }

template <class TX, class TH, int TPR, int NV>
__global__ __launch_bounds__(norm_threads<TPR>()) void rms_norm_kernel(NormArgs p) {
  constexpr int RPB = norm_threads<TPR>() / TPR;
  __shared__ float sums[16];
  __shared__ uint32_t tops[16];
  const int t = threadIdx.x % TPR, H = p.hidden;
  // one round for all but the longest inputs, whose rows pass the launch's limit
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + threadIdx.x / TPR; row < p.rows;
       row += static_cast<int64_t>(gridDim.x) * RPB) {
  if (TPR > 64 && row >= gridDim.x) __syncthreads();  // the round before has read `sums` and `tops`
  float v[NV][8];
  float ss = 0.0f;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = (u * TPR + t) * 8, n = H - c;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
    if (n <= 0) continue;
    load8(static_cast<const TX*>(p.x) + row * p.ldx + c, n, v[u]);
    if (p.res) {
      float r[8];
      TH h[8];
      load8(static_cast<const TH*>(p.res) + row * p.ldr + c, n, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[i] = static_cast<TH>(v[u][i] + r[i]);
        v[u][i] = static_cast<float>(h[i]);
      }
      store8(static_cast<TH*>(p.h) + row * H + c, n, h);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += v[u][i] * v[u][i];
  }
  if (p.norm) {
    const float r = rsqrtf(row_sum<TPR>(ss, sums) / static_cast<float>(H) + p.eps);
    if (p.rstd && t == 0) p.rstd[row] = r;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (u * TPR + t) * 8, n = H - c;
      if (n <= 0) continue;
      float w[8];
      if (p.w) load8_any(p.w, p.w_type, c, n, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] *= p.w ? r * w[i] : r;
    }
  }
  if (p.y_type != MM_T_INT8 && p.y_type != MM_T_E4M3) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (u * TPR + t) * 8, n = H - c;
      if (n > 0) store8_f32(static_cast<TX*>(p.y) + row * H + c, n, v[u]);
    }
    continue;
  }
  // The maximum is taken of the bit patterns: NaN lies above infinity there,
  // so a row that holds either shows it.
  uint32_t top = 0;
#pragma unroll
  for (int u = 0; u < NV; ++u)
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7fffffffu);
  top = row_umax<TPR>(top, tops);
  const float most = p.y_type == MM_T_INT8 ? 127.0f : kFp8Max;
  const bool finite = top < 0x7f800000u;
  const float a = fmaxf(__uint_as_float(top), kScaleFloor);
  const float s = !finite ? __uint_as_float(0x7fc00000u) : top == 0 ? 1.0f : a / most;
  const float inv = finite ? most / a : 0.0f;
  if (t == 0) p.scale[row] = s;
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = (u * TPR + t) * 8, n = H - c;
    if (n <= 0) continue;
    uint8_t q[8];
    if (p.y_type == MM_T_INT8) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        q[i] = finite ? static_cast<uint8_t>(static_cast<int>(__builtin_rintf(v[u][i] * inv))) : 0;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = finite ? static_cast<uint8_t>(f32_to_e4m3fn(v[u][i] * inv)) : 0;
    }
    store8(static_cast<uint8_t*>(p.y) + row * H + c, n, q);
  }
  }
}

// Workgroups take rows in strides of the grid and keep dw's sums of their rows
// in registers; each leaves one row of `partial` (the waves' sums joined
// through LDS in wave order), which dw_sum_kernel adds up. No atomics: the
// order, and with it the result, is fixed by the sizes.
template <class TX, class TH, int TPR, int NV>
__global__ __launch_bounds__(norm_threads<TPR>()) void rms_norm_bwd_kernel(NormBwdArgs p) {
  constexpr int RPB = norm_threads<TPR>() / TPR;
  __shared__ float sums[2][16];
  __shared__ float join[TPR == 64 ? RPB * TPR * NV * 8 : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR, H = p.hidden;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    const int c = (u * TPR + t) * 8, n = H - c;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[u][i] = 1.0f;
      dw[u][i] = 0.0f;
    }
    if (p.w && n > 0) load8_any(p.w, p.w_type, c, n, w[u]);
  }
  int parity = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * RPB + sub; row < p.rows;
       row += static_cast<int64_t>(gridDim.x) * RPB) {
    const float r = p.rstd[row];
    float g[NV][8], h[NV][8];
    float dot = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (u * TPR + t) * 8, n = H - c;
#pragma unroll
      for (int i = 0; i < 8; ++i) g[u][i] = h[u][i] = 0.0f;
      if (n <= 0) continue;
      load8(static_cast<const TX*>(p.dy) + row * p.lddy + c, n, g[u]);
      load8(static_cast<const TH*>(p.h) + row * p.ldh + c, n, h[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dw[u][i] += g[u][i] * (h[u][i] * r);
        g[u][i] *= w[u][i];
        dot += g[u][i] * h[u][i];
      }
    }
    dot = row_sum<TPR>(dot, sums[parity]);
    parity ^= 1;
    const float c1 = r * r * r * (dot / static_cast<float>(H));
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (u * TPR + t) * 8, n = H - c;
      if (n <= 0) continue;
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = r * g[u][i] - h[u][i] * c1;
      if (p.dh) {
        float e[8];
        load8(static_cast<const TH*>(p.dh) + row * p.lddh + c, n, e);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] += e[i];
      }
      store8_f32(static_cast<TX*>(p.dx) + row * H + c, n, d);
      if (p.dres) store8_f32(static_cast<TH*>(p.dres) + row * H + c, n, d);
    }
  }
  if (!p.partial) return;
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * H;
  if constexpr (TPR == 64) {
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) join[(sub * NV + u) * TPR * 8 + t * 8 + i] = dw[u][i];
    __syncthreads();
    for (int c = threadIdx.x; c < H; c += norm_threads<TPR>()) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < RPB; ++k) s += join[k * NV * TPR * 8 + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int c = (u * TPR + t) * 8, n = H - c;
      if (n > 0) store8_f32(out + c, n, dw[u]);
    }
  }
}

// dw[c] = sum over the workgroups' partial rows, in order within each of 16
// interleaved shares and then over the shares.
__global__ __launch_bounds__(1024) void dw_sum_kernel(const float* __restrict__ partial, int parts, int H, int w_type,
                                                      void* __restrict__ dw) {
  __shared__ float lds[16][64];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), share = threadIdx.x >> 6;
  float s = 0.0f;
  if (c < H)
#pragma unroll 8
    for (int i = share; i < parts; i += 16) s += partial[static_cast<int64_t>(i) * H + c];
  lds[share][threadIdx.x & 63] = s;
  __syncthreads();
  if (share || c >= H) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) s += lds[i][threadIdx.x];
  if (w_type == MM_T_FP32)
    static_cast<float*>(dw)[c] = s;
  else if (w_type == MM_T_FP16)
    static_cast<_Float16*>(dw)[c] = static_cast<_Float16>(s);
  else
    static_cast<bf16*>(dw)[c] = static_cast<bf16>(s);
}

constexpr int kMaxHidden = 32768;  // 1024 threads of 4 vectors

// Threads and vectors for a row of H columns.
template <class F>
int by_hidden(int H, F&& f) {
  const int v = (H + 7) / 8;
  if (v <= 64) return f.template operator()<64, 1>();
  if (v <= 128) return f.template operator()<64, 2>();
  if (v <= 256) return f.template operator()<64, 4>();
  if (v <= 512) return f.template operator()<256, 2>();
  if (v <= 1024) return f.template operator()<256, 4>();
  if (v <= 2048) return f.template operator()<1024, 2>();
  return f.template operator()<1024, 4>();
}

template <class TX, class TH>
struct LaunchFwd {
  const NormArgs& p;
  hipStream_t s;
  template <int TPR, int NV>
  int operator()() const {
    constexpr int RPB = norm_threads<TPR>() / TPR;
    const int64_t need = (p.rows + RPB - 1) / RPB, most = (int64_t(1) << 31) / norm_threads<TPR>();
    rms_norm_kernel<TX, TH, TPR, NV>
        <<<static_cast<uint32_t>(need < most ? need : most), norm_threads<TPR>(), 0, s>>>(p);
    return mm_check_launch("rms_norm_kernel");
  }
};

// Workgroups of the backward: four to a CU, which is as many as keep the
// memory busy; more would only lengthen the sum over their partial rows.
constexpr int kBwdGroups = 1024;

template <int TPR>
int bwd_groups(int64_t rows) {
  constexpr int RPB = norm_threads<TPR>() / TPR;
  const int64_t need = (rows + RPB - 1) / RPB, most = kBwdGroups * 256 / norm_threads<TPR>();
  return static_cast<int>(need < most ? need : most);
}

template <class TX, class TH>
struct LaunchBwd {
  const NormBwdArgs& p;
  void* dw;
  hipStream_t s;
  template <int TPR, int NV>
  int operator()() const {
    const int groups = bwd_groups<TPR>(p.rows);
    rms_norm_bwd_kernel<TX, TH, TPR, NV><<<groups, norm_threads<TPR>(), 0, s>>>(p);
    const int rc = mm_check_launch("rms_norm_bwd_kernel");
    if (rc || !dw) return rc;
    dw_sum_kernel<<<(p.hidden + 63) / 64, 1024, 0, s>>>(p.partial, groups, p.hidden, p.w_type, dw);
    return mm_check_launch("dw_sum_kernel");
  }
};

struct CountBwd {
  int64_t rows;
  template <int TPR, int NV>
  int operator()() const { return bwd_groups<TPR>(rows); }
};

bool is_float_type(int t) { return t == MM_T_BF16 || t == MM_T_FP16 || t == MM_T_FP32; }

template <template <class, class> class L, class... A>
int by_types(int x_type, int h_type, int H, const A&... a) {
  if (x_type == MM_T_FP32) return by_hidden(H, L<float, float>{a...});
  if (x_type == MM_T_FP16)
    return h_type == MM_T_FP32 ? by_hidden(H, L<_Float16, float>{a...}) : by_hidden(H, L<_Float16, _Float16>{a...});
  return h_type == MM_T_FP32 ? by_hidden(H, L<bf16, float>{a...}) : by_hidden(H, L<bf16, bf16>{a...});
}

bool rows_ok(int64_t rows) { return rows >= 0 && rows < (int64_t(1) << 31); }

}  // namespace

extern "C" int mm_rms_norm(const void* x, int64_t ldx, int32_t x_type, const void* residual, int64_t ldr,
                           int32_t h_type, const void* weight, int32_t weight_type, int64_t rows, int32_t hidden,
                           float eps, void* h_out, void* y, int32_t y_type, float* scale, float* rstd,
                           mm_stream_t stream) {
  MM_CHECK_ARG(rows_ok(rows) && hidden > 0 && hidden <= kMaxHidden, "mm_rms_norm: bad sizes (rows %lld, hidden %d)",
               static_cast<long long>(rows), hidden);
  MM_CHECK_ARG(is_float_type(x_type) && (h_type == x_type || h_type == MM_T_FP32) && (!weight || is_float_type(weight_type)),
               "mm_rms_norm: bad types");
  const bool eight = y_type == MM_T_INT8 || y_type == MM_T_E4M3;
  MM_CHECK_ARG(eight || y_type == x_type, "mm_rms_norm: the output has the input's type or 8 bits");
  if (rows == 0) return MM_OK;
  MM_CHECK_ARG(x && y && (!residual || h_out) && (!eight || scale), "mm_rms_norm: null pointer");
  const NormArgs p{x, residual, weight, h_out, y, scale, rstd, ldx, ldr, rows, hidden, weight_type, y_type, 1, eps};
  return by_types<LaunchFwd>(x_type, residual ? h_type : x_type, hidden, p, mm_hip_stream(stream));
}

extern "C" int mm_quantize_rows(const void* x, int64_t ldx, int32_t x_type, int64_t rows, int32_t cols, void* q,
                                int32_t q_type, float* scale, mm_stream_t stream) {
  MM_CHECK_ARG(rows_ok(rows) && cols > 0 && cols <= kMaxHidden, "mm_quantize_rows: bad sizes (rows %lld, columns %d)",
               static_cast<long long>(rows), cols);
  MM_CHECK_ARG(is_float_type(x_type) && (q_type == MM_T_INT8 || q_type == MM_T_E4M3), "mm_quantize_rows: bad types");
  if (rows == 0) return MM_OK;
  MM_CHECK_ARG(x && q && scale, "mm_quantize_rows: null pointer");
  const NormArgs p{x, nullptr, nullptr, nullptr, q, scale, nullptr, ldx, 0, rows, cols, 0, q_type, 0, 0.0f};
  return by_types<LaunchFwd>(x_type, x_type, cols, p, mm_hip_stream(stream));
}

extern "C" size_t mm_rms_norm_bwd_workspace_bytes(int64_t rows, int32_t hidden) {
  if (!rows_ok(rows) || hidden <= 0 || hidden > kMaxHidden) return 0;
  return static_cast<size_t>(by_hidden(hidden, CountBwd{rows})) * hidden * 4;
}

extern "C" int mm_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh,
                               const void* weight, int32_t weight_type, const float* rstd, int32_t x_type,
                               int32_t h_type, int64_t rows, int32_t hidden, void* dx, void* dresidual, void* dweight,
                               void* workspace, size_t workspace_bytes, mm_stream_t stream) {
  MM_CHECK_ARG(rows_ok(rows) && hidden > 0 && hidden <= kMaxHidden,
               "mm_rms_norm_bwd: bad sizes (rows %lld, hidden %d)", static_cast<long long>(rows), hidden);
  MM_CHECK_ARG(is_float_type(x_type) && (h_type == x_type || h_type == MM_T_FP32) &&
                   ((!weight && !dweight) || is_float_type(weight_type)),
               "mm_rms_norm_bwd: bad types");
  MM_CHECK_ARG(rows == 0 || (dx && dy && h && rstd), "mm_rms_norm_bwd: null pointer");
  if (dweight && workspace_bytes < mm_rms_norm_bwd_workspace_bytes(rows, hidden)) {
    mm_set_error("mm_rms_norm_bwd: workspace needs %zu bytes", mm_rms_norm_bwd_workspace_bytes(rows, hidden));
    return MM_E_WS;
  }
  MM_CHECK_ARG(!dweight || rows == 0 || workspace, "mm_rms_norm_bwd: null workspace");
  const hipStream_t s = mm_hip_stream(stream);
  if (rows == 0) {  // no rows: the weight's gradient is an empty sum
    if (!dweight) return MM_OK;
    dw_sum_kernel<<<(hidden + 63) / 64, 1024, 0, s>>>(nullptr, 0, hidden, weight_type, dweight);
    return mm_check_launch("dw_sum_kernel");
  }
  const NormBwdArgs p{dy,   dh,   h,   weight, rstd,   dx, dresidual, dweight ? static_cast<float*>(workspace) : nullptr,
                      lddy, lddh, ldh, rows,   hidden, weight_type};
  return by_types<LaunchBwd>(x_type, h_type, hidden, p, dweight, s);
}
