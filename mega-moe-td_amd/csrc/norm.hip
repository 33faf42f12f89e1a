// Root-mean-square norm of rows with the residual's addition, its backward,
// and rows in 8 bits with one scale each.
//
//   h = round(x + residual)          (h = x without a residual)
//   y = h * r * w,  r = 1 / sqrt(mean(h^2) + eps)
//   8 bits: s = max(a, 1e-30) / Q with a = max |y| over the row (s = 1 where
//           a = 0), q = round(y / s) of the unrounded y; Q = 127 (int8) or 448 (E4M3)
//   backward, with n = h r: dx = dh + r (w dy - n mean(w dy n)),  dw = sum_rows dy n
//           (n is near 1 whatever the row's size; r^3 would leave fp32 from rows
//           of 1e13 on)
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

// A mean square that fp32 cannot hold, from rows of 1e19 / sqrt(H) on or, with an
// eps as small, of 1e-15 and below: the row is multiplied by a power of two,
// which leaves y as it is, and summed again. 2^-74 brings the largest row's sum
// below the largest fp32 and 2^100 the smallest row's above the smallest. Rare,
// and the same for all threads of a row.
__device__ __forceinline__ bool out_of_range(float mean_square) {
  return !(mean_square >= 0x1p-100f && mean_square < __builtin_inff());
}
__device__ __forceinline__ float into_range(float mean_square) { return mean_square < 1.0f ? 0x1p100f : 0x1p-74f; }

// Eight consecutive elements as they lie in memory, at any alignment of their
// type (one or two 16-byte loads). Loads stay apart from the conversions, so
// that all of a row's are in flight before the first is needed: converting each
// where it is loaded, inside the branch that cuts the row's end, cost 30%
// (8192 x 2048 with a residual, 43 us against 30).
template <class T>
struct Vec8 {
  T v[8];
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    __builtin_memcpy(v, static_cast<const T*>(p) + at, sizeof(v));
  }
  __device__ __forceinline__ void store(void* p, int64_t at) const {
    __builtin_memcpy(static_cast<T*>(p) + at, v, sizeof(v));
  }
  __device__ __forceinline__ void to_f32(float* f) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(v[i]);
  }
  __device__ __forceinline__ static Vec8 of(const float* f) {
    Vec8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = static_cast<T>(f[i]);
    return r;
  }
};

// The weight's vector, of a type known at run time.
struct WeightVec8 {
  uint32_t raw[8];
  __device__ __forceinline__ void load(const void* p, int type, int at) {
    if (type == MM_T_FP32)
      __builtin_memcpy(raw, static_cast<const float*>(p) + at, 32);
    else
      __builtin_memcpy(raw, static_cast<const uint16_t*>(p) + at, 16);
  }
  __device__ __forceinline__ void to_f32(int type, float* f) const {
    if (type == MM_T_FP32) {
      __builtin_memcpy(f, raw, 32);
    } else if (type == MM_T_FP16) {
      Vec8<_Float16> h;
      __builtin_memcpy(h.v, raw, 16);
      h.to_f32(f);
    } else {
      Vec8<bf16> h;
      __builtin_memcpy(h.v, raw, 16);
      h.to_f32(f);
    }
  }
};

// Columns of vector i of a row. The last one of a row whose length is no
// multiple of 8 is moved to the row's end: the columns it shares with the one
// before are computed twice with one value, and counted in a sum once.
struct Columns {
  int at, own;  // first column; the first that this vector counts (8 or more: none)
  __device__ __forceinline__ Columns(int i, int H) : at(min(i * 8, H - 8)), own(i * 8 - at) {}
  __device__ __forceinline__ bool any() const { return own < 8; }
  __device__ __forceinline__ bool counts(int i) const { return i >= own; }
};

__device__ __forceinline__ float load_any(const void* p, int type, int at) {
  if (type == MM_T_FP32) return static_cast<const float*>(p)[at];
  if (type == MM_T_FP16) return static_cast<float>(static_cast<const _Float16*>(p)[at]);
  return static_cast<float>(static_cast<const bf16*>(p)[at]);
}

// A row belongs to one wave (WAVE: 4 rows a workgroup, no barriers) or to the
// whole workgroup; its threads hold NV vectors each, thread t the vectors t,
// t + threads, ... Reductions give every thread of the row the result. `lds`
// has one slot a wave; successive calls alternate between two such arrays, so
// a slot is rewritten only behind a later call's barrier.
constexpr int kWaveThreads = 256, kWaveRows = kWaveThreads / 64;

template <bool WAVE>
__device__ __forceinline__ float row_sum(float v, float* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
    for (int i = 0; i < static_cast<int>(blockDim.x / 64); ++i) v += lds[i];
  }
  return v;
}

template <bool WAVE>
__device__ __forceinline__ uint32_t row_umax(uint32_t v, uint32_t* lds) {
#pragma unroll
  for (int m = 32; m > 0; m >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), m)));
  if constexpr (!WAVE) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int i = 0; i < static_cast<int>(blockDim.x / 64); ++i) v = max(v, lds[i]);
  }
  return v;
}

// Rows in 8 bits. r = mant * pow2 with 1 <= mant < 2, and a row's values are
// held as t = h pow2 w = y / mant: for 16-bit h and w that is exact, and mant
// drops out of the quotient y / s = t Q / max |t|. Quotients that lie on a
// rounding border exactly, about 1 in 10^4 of them, thus come out exact and
// round to even; a rounded y would send them either way.
struct Rsqrt {
  float mant, pow2;
  __device__ __forceinline__ explicit Rsqrt(float r)  // of 0 and infinity: 1 and itself
      : mant(__uint_as_float((__float_as_uint(r) & 0x007fffffu) | 0x3f800000u)),
        pow2(__uint_as_float(__float_as_uint(r) & 0x7f800000u)) {}
};

struct Quantizer {
  float top, most, inv, fix, scale;
  bool finite;
  // bits: largest |t| as a bit pattern, where NaN lies above infinity, so that a
  // row that holds either shows it
  __device__ __forceinline__ Quantizer(uint32_t bits, float mant, bool e4m3) : top(__uint_as_float(bits)) {
    const float q = e4m3 ? kFp8Max : 127.0f, a = top * mant;
    const bool small = a < kScaleFloor, large = top > 1e30f;  // Q / top, t Q would leave the range
    finite = a < __builtin_inff();
    most = large ? 1.0f : q;
    inv = small ? mant / kScaleFloor : large ? q / top : 1.0f / top;
    fix = small || large ? 0.0f : inv;
    scale = !finite ? __uint_as_float(0x7fc00000u) : bits == 0 ? 1.0f : fmaxf(a, kScaleFloor) / q;
  }
  // t Q / top: one correction of the quotient makes it exact where it is
  // representable, with what t Q loses to rounding (22 bits of fp16 products and
  // 7 of Q). |value| stays below the border of the largest, so neither
  // type saturates.
  __device__ __forceinline__ float value(float t) const {
    const float p = t * most, rest = fmaf(t, most, -p), q = p * inv;
    return fmaf(fmaf(-q, top, p) + rest, fix, q);
  }
};

// 8 values into int8 or E4M3, round to nearest even.
__device__ __forceinline__ uint2 quantize8(const float* v, const Quantizer& z, bool e4m3) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = z.value(v[4 * h + i]);
    if (e4m3) {
      int d = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
      w[h] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], d, true));
    } else {
      w[h] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[h] |= (static_cast<uint32_t>(static_cast<int>(__builtin_rintf(s[i]))) & 0xffu) << (8 * i);
    }
  }
  return make_uint2(w[0], w[1]);
}

// Two vectors of 16 bits a thread fit the registers of six waves, which the
// compiler misses by two of them by itself (8192 x 7168: 94 us, 87 so).
template <class TX, class TH, int NV, bool WAVE>
__global__ __launch_bounds__(WAVE ? kWaveThreads : 1024)
__attribute__((amdgpu_waves_per_eu(!WAVE && NV == 2 && sizeof(TX) + sizeof(TH) == 4 ? 6 : 4))) void rms_norm_kernel(NormArgs p) {
  __shared__ float sums[16];
  __shared__ uint32_t tops[16];
  const int threads = WAVE ? 64 : blockDim.x, t = WAVE ? threadIdx.x & 63 : threadIdx.x, H = p.hidden;
  const int64_t first = WAVE ? static_cast<int64_t>(blockIdx.x) * kWaveRows + (threadIdx.x >> 6) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WAVE ? kWaveRows : 1);
  // one round for all but the longest inputs, whose rows pass the launch's limit
  for (int64_t row = first; row < p.rows; row += step) {
    if (!WAVE && row != first) __syncthreads();  // the row before has been read from `sums` and `tops`
    Vec8<TX> x[NV];
    Vec8<TH> res[NV];
    WeightVec8 wv[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) x[u].load(p.x, row * p.ldx + Columns(u * threads + t, H).at);
    if (p.res)
#pragma unroll
      for (int u = 0; u < NV; ++u) res[u].load(p.res, row * p.ldr + Columns(u * threads + t, H).at);
    if (p.w)
#pragma unroll
      for (int u = 0; u < NV; ++u) wv[u].load(p.w, p.w_type, Columns(u * threads + t, H).at);
    float v[NV][8];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      x[u].to_f32(v[u]);
      if (p.res) {
        const Columns c(u * threads + t, H);
        float r[8];
        res[u].to_f32(r);
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] += v[u][i];
        const Vec8<TH> h = Vec8<TH>::of(r);
        if (c.any()) h.store(p.h, row * H + c.at);
        h.to_f32(v[u]);
      }
    }
    const bool eight = p.y_type == MM_T_INT8 || p.y_type == MM_T_E4M3;
    float mant = 1.0f;
    if (p.norm) {
      float mean, k = 1.0f;
#pragma clang loop unroll(disable)  // a second copy of the sum costs registers (99 us instead of 87)
      for (;;) {
        float ss = 0.0f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          const Columns c(u * threads + t, H);
#pragma unroll
          for (int i = 0; i < 8; ++i) ss += c.counts(i) ? v[u][i] * v[u][i] : 0.0f;
        }
        mean = row_sum<WAVE>(ss, sums) / static_cast<float>(H) + p.eps * k * k;
        if (k != 1.0f || !out_of_range(mean)) break;
        k = into_range(mean);
#pragma unroll
        for (int u = 0; u < NV; ++u)
#pragma unroll
          for (int i = 0; i < 8; ++i) v[u][i] *= k;
        if (!WAVE) __syncthreads();  // the sum has been read from `sums`
      }
      float r = rsqrtf(mean);
      if (p.rstd && t == 0) p.rstd[row] = r * k;
      if (eight) {
        const Rsqrt split(r);
        mant = split.mant;
        r = split.pow2;
      }
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float w[8];
        if (p.w) wv[u].to_f32(p.w_type, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] *= p.w ? r * w[i] : r;
      }
    }
    if (!eight) {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const Columns c(u * threads + t, H);
        if (c.any()) Vec8<TX>::of(v[u]).store(p.y, row * H + c.at);
      }
      continue;
    }
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[u][i]) & 0x7fffffffu);
    const bool e4m3 = p.y_type == MM_T_E4M3;
    const Quantizer z(row_umax<WAVE>(top, tops), mant, e4m3);
    if (t == 0) p.scale[row] = z.scale;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const Columns c(u * threads + t, H);
      const uint2 q = z.finite ? quantize8(v[u], z, e4m3) : make_uint2(0, 0);
      if (c.any()) __builtin_memcpy(static_cast<uint8_t*>(p.y) + row * H + c.at, &q, 8);
    }
  }
}

// Rows of fewer than 8 columns: a thread has a row.
template <class TX, class TH>
__global__ __launch_bounds__(256) void rms_norm_short_kernel(NormArgs p) {
  const int H = p.hidden;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; row < p.rows;
       row += static_cast<int64_t>(gridDim.x) * 256) {
    float v[8], ss = 0.0f;
    for (int i = 0; i < H; ++i) {
      v[i] = static_cast<float>(static_cast<const TX*>(p.x)[row * p.ldx + i]);
      if (p.res) {
        const TH h = static_cast<TH>(v[i] + static_cast<float>(static_cast<const TH*>(p.res)[row * p.ldr + i]));
        static_cast<TH*>(p.h)[row * H + i] = h;
        v[i] = static_cast<float>(h);
      }
      ss += v[i] * v[i];
    }
    const bool eight = p.y_type == MM_T_INT8 || p.y_type == MM_T_E4M3;
    float mant = 1.0f;
    if (p.norm) {
      float mean = ss / static_cast<float>(H) + p.eps, k = 1.0f;
      if (out_of_range(mean)) {
        k = into_range(mean);
        ss = 0.0f;
        for (int i = 0; i < H; ++i) {
          v[i] *= k;
          ss += v[i] * v[i];
        }
        mean = ss / static_cast<float>(H) + p.eps * k * k;
      }
      float r = rsqrtf(mean);
      if (p.rstd) p.rstd[row] = r * k;
      if (eight) {
        const Rsqrt split(r);
        mant = split.mant;
        r = split.pow2;
      }
      for (int i = 0; i < H; ++i) v[i] *= p.w ? r * load_any(p.w, p.w_type, i) : r;
    }
    if (!eight) {
      for (int i = 0; i < H; ++i) static_cast<TX*>(p.y)[row * H + i] = static_cast<TX>(v[i]);
      continue;
    }
    uint32_t top = 0;
    for (int i = 0; i < 8; ++i) {
      if (i >= H) v[i] = 0.0f;
      top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    const bool e4m3 = p.y_type == MM_T_E4M3;
    const Quantizer z(top, mant, e4m3);
    p.scale[row] = z.scale;
    const uint2 q = z.finite ? quantize8(v, z, e4m3) : make_uint2(0, 0);
    for (int i = 0; i < H; ++i)
      static_cast<uint8_t*>(p.y)[row * H + i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

// Workgroups take rows in strides of the grid and keep dw's sums of their rows
// in registers; each leaves one row of `partial` (the waves' sums joined
// through LDS in wave order), which dw_sum_kernel adds up. No atomics: the
// order, and with it the result, is fixed by the sizes.
template <class TX, class TH, int NV, bool WAVE>
__global__ __launch_bounds__(WAVE ? kWaveThreads : 1024) void rms_norm_bwd_kernel(NormBwdArgs p) {
  __shared__ float sums[2][16];
  __shared__ float join[WAVE ? kWaveRows * 64 * NV * 8 : 1];
  const int threads = WAVE ? 64 : blockDim.x, t = WAVE ? threadIdx.x & 63 : threadIdx.x, H = p.hidden;
  const int sub = WAVE ? threadIdx.x >> 6 : 0, rpb = WAVE ? kWaveRows : 1;
  float w[NV][8], dw[NV][8];
#pragma unroll
  for (int u = 0; u < NV; ++u) {
    WeightVec8 wv;
    if (p.w) wv.load(p.w, p.w_type, Columns(u * threads + t, H).at);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      w[u][i] = 1.0f;
      dw[u][i] = 0.0f;
    }
    if (p.w) wv.to_f32(p.w_type, w[u]);
  }
  int parity = 0;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * rpb + sub; row < p.rows;
       row += static_cast<int64_t>(gridDim.x) * rpb) {
    const float r = p.rstd[row];  // first, as the dot product waits for it (8192 x 2048: 29 us behind the rows, 26 so)
    Vec8<TX> gv[NV];
    Vec8<TH> hv[NV], ev[NV];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int at = Columns(u * threads + t, H).at;
      gv[u].load(p.dy, row * p.lddy + at);
      hv[u].load(p.h, row * p.ldh + at);
    }
    if (p.dh)
#pragma unroll
      for (int u = 0; u < NV; ++u) ev[u].load(p.dh, row * p.lddh + Columns(u * threads + t, H).at);
    float g[NV][8], h[NV][8];
    float dot = 0.0f;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const Columns c(u * threads + t, H);
      gv[u].to_f32(g[u]);
      hv[u].to_f32(h[u]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        h[u][i] *= r;
        dw[u][i] += g[u][i] * h[u][i];
        g[u][i] *= w[u][i];
        dot += c.counts(i) ? g[u][i] * h[u][i] : 0.0f;
      }
    }
    dot = row_sum<WAVE>(dot, sums[parity]);
    parity ^= 1;
    const float mean = dot / static_cast<float>(H);
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const Columns c(u * threads + t, H);
      float d[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) d[i] = r * (g[u][i] - h[u][i] * mean);
      if (p.dh) {
        float e[8];
        ev[u].to_f32(e);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] += e[i];
      }
      if (c.any()) {
        Vec8<TX>::of(d).store(p.dx, row * H + c.at);
        if (p.dres) Vec8<TH>::of(d).store(p.dres, row * H + c.at);
      }
    }
  }
  if (!p.partial) return;
  float* out = p.partial + static_cast<int64_t>(blockIdx.x) * H;
  if constexpr (WAVE) {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const Columns c(u * 64 + t, H);
      if (c.any()) __builtin_memcpy(join + sub * 512 * NV + c.at, dw[u], 32);
    }
    __syncthreads();
    for (int c = threadIdx.x; c < H; c += kWaveThreads) {
      float s = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaveRows; ++k) s += join[k * 512 * NV + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const Columns c(u * threads + t, H);
      if (c.any()) __builtin_memcpy(out + c.at, dw[u], 32);
    }
  }
}

// Rows of fewer than 8 columns: a thread has a row at a time; the workgroup's
// threads are joined column by column.
template <class TX, class TH>
__global__ __launch_bounds__(256) void rms_norm_short_bwd_kernel(NormBwdArgs p) {
  __shared__ float join[256];
  const int H = p.hidden;
  float w[8], dw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = p.w && i < H ? load_any(p.w, p.w_type, i) : 1.0f;
    dw[i] = 0.0f;
  }
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; row < p.rows;
       row += static_cast<int64_t>(gridDim.x) * 256) {
    const float r = p.rstd[row];
    float g[8], h[8], dot = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g[i] = i < H ? static_cast<float>(static_cast<const TX*>(p.dy)[row * p.lddy + i]) : 0.0f;
      h[i] = i < H ? static_cast<float>(static_cast<const TH*>(p.h)[row * p.ldh + i]) * r : 0.0f;
      dw[i] += g[i] * h[i];
      g[i] *= w[i];
      dot += g[i] * h[i];
    }
    const float mean = dot / static_cast<float>(H);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= H) continue;
      float d = r * (g[i] - h[i] * mean);
      if (p.dh) d += static_cast<float>(static_cast<const TH*>(p.dh)[row * p.lddh + i]);
      static_cast<TX*>(p.dx)[row * H + i] = static_cast<TX>(d);
      if (p.dres) static_cast<TH*>(p.dres)[row * H + i] = static_cast<TH>(d);
    }
  }
  if (!p.partial) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    __syncthreads();
    join[threadIdx.x] = dw[i];
    __syncthreads();
    for (int m = 128; m > 0; m >>= 1) {
      if (static_cast<int>(threadIdx.x) < m) join[threadIdx.x] += join[threadIdx.x + m];
      __syncthreads();
    }
    if (threadIdx.x == 0 && i < H) p.partial[static_cast<int64_t>(blockIdx.x) * H + i] = join[0];
  }
}

// dw[c] = sum over the workgroups' partial rows, in order within each of 32
// interleaved shares and then over the shares. A share reads a line of 32
// columns: with 64 columns and 16 shares, half as many workgroups, 1024 partial
// rows of 2048 columns took 4.7 us, so 4.0.
constexpr int kSumColumns = 32, kShares = 1024 / kSumColumns;
__global__ __launch_bounds__(1024) void dw_sum_kernel(const float* __restrict__ partial, int parts, int H, int w_type,
                                                      void* __restrict__ dw) {
  __shared__ float lds[kShares][kSumColumns];
  const int c = blockIdx.x * kSumColumns + threadIdx.x % kSumColumns, share = threadIdx.x / kSumColumns;
  float s = 0.0f;
  if (c < H)
    for (int i = share; i < parts; i += 8 * kShares) {  // 8 rows in flight, also the last
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        v[u] = i + u * kShares < parts ? partial[static_cast<int64_t>(i + u * kShares) * H + c] : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
  lds[share][threadIdx.x % kSumColumns] = s;
  __syncthreads();
  if (share || c >= H) return;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < kShares; ++i) s += lds[i][threadIdx.x];
  if (w_type == MM_T_FP32)
    static_cast<float*>(dw)[c] = s;
  else if (w_type == MM_T_FP16)
    static_cast<_Float16*>(dw)[c] = static_cast<_Float16>(s);
  else
    static_cast<bf16*>(dw)[c] = static_cast<bf16>(s);
}

constexpr int kMaxHidden = 32768;  // 1024 threads of 4 vectors

// How a row of H columns is held: NV vectors a thread, by a wave or by a
// workgroup of `threads`. One vector a thread is fastest as far as it goes (8192
// x 2048 forward: 24 us, two 25, four in a wave 47) until a workgroup takes
// half a CU (7168 columns: 118 us with one, 92 with two). The backward keeps
// short rows in waves, 4 to a workgroup, so that few partial sums are left
// (16384 x 1024: 24 us + 4 for their sum, in workgroups 27 + 7).
template <bool BACKWARD, class F>
int by_hidden(int H, F&& f) {
  if (H < 8) return f.short_rows();
  const int v = (H + 7) / 8;
  auto threads = [&](int nv) { return (v + 64 * nv - 1) / (64 * nv) * 64; };
  if (v <= 64) return f.template operator()<1, true>(64);
  if constexpr (BACKWARD) {
    if (v <= 128) return f.template operator()<2, true>(64);
  }
  if (v <= 512) return f.template operator()<1, false>(threads(1));
  if (v <= 2048) return f.template operator()<2, false>(threads(2));
  return f.template operator()<4, false>(threads(4));
}

template <class TX, class TH>
struct LaunchFwd {
  const NormArgs& p;
  hipStream_t s;
  template <int NV, bool WAVE>
  int operator()(int threads) const {
    const int size = WAVE ? kWaveThreads : threads, rpb = WAVE ? kWaveRows : 1;
    const int64_t need = (p.rows + rpb - 1) / rpb, most = (int64_t(1) << 31) / size;
    rms_norm_kernel<TX, TH, NV, WAVE><<<static_cast<uint32_t>(need < most ? need : most), size, 0, s>>>(p);
    return mm_check_launch("rms_norm_kernel");
  }
  int short_rows() const {
    const int64_t need = (p.rows + 255) / 256;
    rms_norm_short_kernel<TX, TH><<<static_cast<uint32_t>(need < 65536 ? need : 65536), 256, 0, s>>>(p);
    return mm_check_launch("rms_norm_short_kernel");
  }
};

// Workgroups of the backward: 16 waves of one vector a CU, or 8 of two, keep
// the memory busy; more would only lengthen the sum over their partial rows
// (8192 x 2048, one vector: 26 + 4 us, with half as many 31 + 4; 16384 x 1024,
// two: 26 + 4, with twice as many 30 + 4). All take equally many rows, so that
// none leaves a partial row for fewer (1021 x 2305: 511 workgroups of 2 rows
// 10.2 + 4.0 us, 819 of 1 or 2 rows 10.9 + 4.9). Workgroups of 8 waves and more
// then leave CUs idle: 128 of them at 16384 columns, 64 at 32768 (2048 x 16384
// with a residual 63 us, 4.2 TB/s; 1024 x 32768 431, with spilled registers).
template <int NV, bool WAVE>
int bwd_groups(int64_t rows, int threads) {
  const int rpb = WAVE ? kWaveRows : 1, waves = (WAVE ? kWaveThreads : threads) / 64;
  const int64_t need = (rows + rpb - 1) / rpb, most = 4096 / NV / waves;
  const int64_t each = need > most ? (need + most - 1) / most : 1;
  return static_cast<int>((need + each - 1) / each);
}

int short_bwd_groups(int64_t rows) { return static_cast<int>((rows + 255) / 256 < 256 ? (rows + 255) / 256 : 256); }

template <class TX, class TH>
struct LaunchBwd {
  const NormBwdArgs& p;
  void* dw;
  hipStream_t s;
  template <int NV, bool WAVE>
  int operator()(int threads) const {
    const int groups = bwd_groups<NV, WAVE>(p.rows, threads);
    rms_norm_bwd_kernel<TX, TH, NV, WAVE><<<groups, WAVE ? kWaveThreads : threads, 0, s>>>(p);
    return add_up(groups);
  }
  int short_rows() const {
    const int groups = short_bwd_groups(p.rows);
    rms_norm_short_bwd_kernel<TX, TH><<<groups, 256, 0, s>>>(p);
    return add_up(groups);
  }
  int add_up(int groups) const {
    const int rc = mm_check_launch("rms_norm_bwd_kernel");
    if (rc || !dw) return rc;
    dw_sum_kernel<<<(p.hidden + kSumColumns - 1) / kSumColumns, 1024, 0, s>>>(p.partial, groups, p.hidden, p.w_type, dw);
    return mm_check_launch("dw_sum_kernel");
  }
};

struct CountBwd {
  int64_t rows;
  template <int NV, bool WAVE>
  int operator()(int threads) const { return bwd_groups<NV, WAVE>(rows, threads); }
  int short_rows() const { return short_bwd_groups(rows); }
};

bool is_float_type(int t) { return t == MM_T_BF16 || t == MM_T_FP16 || t == MM_T_FP32; }

template <bool BACKWARD, template <class, class> class L, class... A>
int by_types(int x_type, int h_type, int H, const A&... a) {
  if (x_type == MM_T_FP32) return by_hidden<BACKWARD>(H, L<float, float>{a...});
  if (x_type == MM_T_FP16)
    return h_type == MM_T_FP32 ? by_hidden<BACKWARD>(H, L<_Float16, float>{a...})
                               : by_hidden<BACKWARD>(H, L<_Float16, _Float16>{a...});
  return h_type == MM_T_FP32 ? by_hidden<BACKWARD>(H, L<bf16, float>{a...})
                             : by_hidden<BACKWARD>(H, L<bf16, bf16>{a...});
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
  return by_types<false, LaunchFwd>(x_type, residual ? h_type : x_type, hidden, p, mm_hip_stream(stream));
}

extern "C" int mm_quantize_rows(const void* x, int64_t ldx, int32_t x_type, int64_t rows, int32_t cols, void* q,
                                int32_t q_type, float* scale, mm_stream_t stream) {
  MM_CHECK_ARG(rows_ok(rows) && cols > 0 && cols <= kMaxHidden, "mm_quantize_rows: bad sizes (rows %lld, columns %d)",
               static_cast<long long>(rows), cols);
  MM_CHECK_ARG(is_float_type(x_type) && (q_type == MM_T_INT8 || q_type == MM_T_E4M3), "mm_quantize_rows: bad types");
  if (rows == 0) return MM_OK;
  MM_CHECK_ARG(x && q && scale, "mm_quantize_rows: null pointer");
  const NormArgs p{x, nullptr, nullptr, nullptr, q, scale, nullptr, ldx, 0, rows, cols, 0, q_type, 0, 0.0f};
  return by_types<false, LaunchFwd>(x_type, x_type, cols, p, mm_hip_stream(stream));
}

extern "C" size_t mm_rms_norm_bwd_workspace_bytes(int64_t rows, int32_t hidden) {
  if (!rows_ok(rows) || hidden <= 0 || hidden > kMaxHidden) return 0;
  return static_cast<size_t>(by_hidden<true>(hidden, CountBwd{rows})) * hidden * 4;
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
    dw_sum_kernel<<<(hidden + kSumColumns - 1) / kSumColumns, 1024, 0, s>>>(nullptr, 0, hidden, weight_type, dweight);
    return mm_check_launch("dw_sum_kernel");
  }
  const NormBwdArgs p{dy,   dh,   h,   weight, rstd,   dx, dresidual, dweight ? static_cast<float*>(workspace) : nullptr,
                      lddy, lddh, ldh, rows,   hidden, weight_type};
  return by_types<true, LaunchBwd>(x_type, h_type, hidden, p, dweight, s);
}
