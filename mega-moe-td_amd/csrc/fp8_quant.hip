// Blocks of 128 values in E4M3 with a power-of-two scale each (fp8.h): rows in
// blocks of 128 columns, matrices in blocks of 128 x 128, and the transposed
// forms that a training step's gradients read.
//
// Memory bound: every value is read once and its byte written once in each
// form that is asked for. 8192 x 7168 in rows: 36 us, 4.85 TB/s of reads and
// writes, a copy's rate; 8192 x 4096 in both forms with a scale for each row and
// column 28 us, 4.8 TB/s, with one for 128 x 128 23 us.
#include "fp8.h"

namespace {

struct QuantArgs {
  const void* x;
  const uint8_t* x_scale;  // E4M3 input: [rows, column blocks]
  uint8_t* q;              // [batch, rows, ldq], or NULL
  uint8_t* scale;          // [batch, row blocks, column blocks]
  uint8_t* qt;             // [cols, ldqt], or NULL
  uint8_t* scale_t;        // [column blocks or cols, row blocks]
  int64_t ldx, x_batch, ldq, ldqt;
  uint32_t batch, rows, cols, kb;  // kb: column blocks
  uint64_t units;                  // batch * rows * kb
};

// Eight consecutive columns of a row in fp32; those from `left` on are 0 and
// not touched.
template <class T>
__device__ __forceinline__ void load8(const T* p, int left, float (&v)[8]) {
  T raw[8];
  if (left >= 8) {
    __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(raw[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? static_cast<float>(p[i]) : 0.0f;
  }
}

__device__ __forceinline__ void store8(uint8_t* p, int left, uint2 w) {
  if (left >= 8) {
    __builtin_memcpy(p, &w, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = static_cast<uint8_t>((i < 4 ? w.x : w.y) >> (8 * (i & 3)));
  }
}

__device__ __forceinline__ uint32_t top8(const float (&v)[8]) {
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) t = max(t, abs_bits(v[i]));
  return t;
}

// A block of 128 columns belongs to 16 lanes.
template <class T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(QuantArgs p) {
  constexpr int U = 4;  // blocks of a lane, all loaded before the first is needed
  const int lane = threadIdx.x & 15;
  const uint64_t first = static_cast<uint64_t>(blockIdx.x) * (16 * U) + (threadIdx.x >> 4);
  float v[U][8];
  uint32_t row[U];
  int col[U];
  bool live[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint64_t unit = first + u * 16;
    live[u] = unit < p.units;
    const uint32_t n = static_cast<uint32_t>(live[u] ? unit : 0);  // units < 2^32
    row[u] = n / p.kb;
    col[u] = static_cast<int>((n - row[u] * p.kb) * kBlock) + lane * 8;
    const uint32_t b = p.batch == 1 ? 0 : row[u] / p.rows;
    load8(static_cast<const T*>(p.x) + b * p.x_batch + static_cast<int64_t>(row[u] - b * p.rows) * p.ldx + col[u],
          static_cast<int>(p.cols) - col[u], v[u]);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const BlockScale s(max16(top8(v[u])));
    if (!live[u]) continue;
    if (lane == 0) p.scale[static_cast<uint64_t>(row[u]) * p.kb + col[u] / kBlock] = static_cast<uint8_t>(s.byte);
    store8(p.q + row[u] * p.ldq + col[u], static_cast<int>(p.ldq) - col[u],
           make_uint2(s.pack4(v[u][0], v[u][1], v[u][2], v[u][3]), s.pack4(v[u][4], v[u][5], v[u][6], v[u][7])));
  }
}

struct E4m3 {
  uint8_t v;
};

// Input values of a tile's row from E4M3 and the scale of their 128 columns.
__device__ __forceinline__ void load8(const E4m3* p, int left, float scale, float (&v)[8]) {
  uint32_t w[2] = {0, 0};
  if (left >= 8) {
    __builtin_memcpy(w, p, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) w[i >> 2] |= static_cast<uint32_t>(p[i].v) << (8 * (i & 3));
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[h]), false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w[h]), true);
    v[4 * h] = lo[0] * scale;
    v[4 * h + 1] = lo[1] * scale;
    v[4 * h + 2] = hi[0] * scale;
    v[4 * h + 3] = hi[1] * scale;
  }
  // a NaN scale marks its columns only
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i >= left) v[i] = 0.0f;
}

// The larger of a value over the four rows of a wave.
__device__ __forceinline__ uint32_t over_rows(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 16)));
  return max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), 32)));
}

// A 128 x 128 tile: 16 lanes hold a row, 8 columns each, and one of NT threads
// 2048 / NT rows. BLOCK: one scale for the tile, in both forms. Otherwise a scale for
// each row in q and for each column in qt. Bytes past the last row are 0 in qt
// (they are summed over), those past the last column 0 in q.
template <class T, bool BLOCK, int NT>
__global__ __launch_bounds__(NT) void quantize_tile_kernel(QuantArgs p) {
  constexpr int U = 2048 / NT, ROWS = NT / 16, W = NT / 64;
  __shared__ uint32_t bytes[128][33];  // a column more, so that a pass over rows spreads over the banks
  __shared__ uint32_t tops[W][BLOCK ? 1 : 128];
  __shared__ __attribute__((aligned(16))) float inverse[BLOCK ? 1 : 128];  // of a column's scale; 0 where a value is not finite
  const int wave = threadIdx.x >> 6;
  const int lane = threadIdx.x & 15, r = threadIdx.x >> 4;
  const uint32_t rb = (p.rows + 127) / 128;  // row blocks
  const uint32_t tile = blockIdx.x % (rb * p.kb), b = blockIdx.x / (rb * p.kb);
  const uint32_t r0 = tile / p.kb * 128, c0 = tile % p.kb * 128;
  const int col = static_cast<int>(c0) + lane * 8, left = static_cast<int>(p.cols) - col;
  float v[U][8];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t row = r0 + u * ROWS + r;
    const int have = row < p.rows ? left : 0;
    const T* x = static_cast<const T*>(p.x) + b * p.x_batch + static_cast<int64_t>(min(row, p.rows - 1)) * p.ldx + col;
    if constexpr (sizeof(T) == 1)
      load8(x, have, scale_value(row < p.rows ? p.x_scale[static_cast<uint64_t>(row) * p.kb + c0 / 128] : 127), v[u]);
    else
      load8(x, have, v[u]);
  }
  uint8_t* const q = p.q ? p.q + static_cast<uint64_t>(b) * p.rows * p.ldq : nullptr;
  uint2 w[U];
  if constexpr (BLOCK) {
    uint32_t top = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) top = max(top, top8(v[u]));
    top = over_rows(max16(top));
    if ((threadIdx.x & 63) == 0) tops[wave][0] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max(top, tops[i][0]);
    const BlockScale s(top);
    if (threadIdx.x == 0) {
      if (p.q) p.scale[(static_cast<uint64_t>(b) * rb + r0 / 128) * p.kb + c0 / 128] = static_cast<uint8_t>(s.byte);
      if (p.qt) p.scale_t[static_cast<uint64_t>(c0 / 128) * rb + r0 / 128] = static_cast<uint8_t>(s.byte);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      w[u] = make_uint2(s.pack4(v[u][0], v[u][1], v[u][2], v[u][3]), s.pack4(v[u][4], v[u][5], v[u][6], v[u][7]));
  }
  if (q) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t row = r0 + u * ROWS + r;
      uint2 o = w[u];
      if constexpr (!BLOCK) {
        const BlockScale s(max16(top8(v[u])));
        o = make_uint2(s.pack4(v[u][0], v[u][1], v[u][2], v[u][3]), s.pack4(v[u][4], v[u][5], v[u][6], v[u][7]));
        if (row < p.rows && lane == 0) p.scale[static_cast<uint64_t>(row) * p.kb + c0 / 128] = static_cast<uint8_t>(s.byte);
      }
      if (row < p.rows) store8(q + row * p.ldq + col, static_cast<int>(p.ldq) - col, o);
    }
  }
  if (!p.qt) return;
  if constexpr (!BLOCK) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t top = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) top = max(top, abs_bits(v[u][i]));
      top = over_rows(top);
      if ((threadIdx.x & 63) < 16) tops[wave][lane * 8 + i] = top;
    }
    __syncthreads();
    if (const uint32_t c = threadIdx.x; c < 128) {
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < W; ++k) top = max(top, tops[k][c]);
      const BlockScale s(top);
      inverse[c] = s.inv;
      if (c0 + c < p.cols) p.scale_t[static_cast<uint64_t>(c0 + c) * rb + r0 / 128] = static_cast<uint8_t>(s.byte);
    }
    __syncthreads();
    float inv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) inv[i] = inverse[lane * 8 + i];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      uint32_t h[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = inv[4 * k + i] == 0.0f ? 0.0f : v[u][4 * k + i] * inv[4 * k + i];
        const int d = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
        h[k] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], d, true));
      }
      w[u] = make_uint2(h[0], h[1]);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    bytes[u * ROWS + r][lane * 2] = w[u].x;
    bytes[u * ROWS + r][lane * 2 + 1] = w[u].y;
  }
  __syncthreads();
  // four rows and four columns at a time; 32 neighbouring lanes write 128 bytes of a column
  const int rq = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 1024 / NT; ++i) {
    const int cq = i * (NT / 32) + (threadIdx.x >> 5);
    uint32_t d[4], o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) d[k] = bytes[rq * 4 + k][cq];
    const uint32_t a = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), c = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u);
    const uint32_t e = __builtin_amdgcn_perm(d[1], d[0], 0x07030602u), f = __builtin_amdgcn_perm(d[3], d[2], 0x07030602u);
    o[0] = __builtin_amdgcn_perm(c, a, 0x05040100u);
    o[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    o[2] = __builtin_amdgcn_perm(f, e, 0x05040100u);
    o[3] = __builtin_amdgcn_perm(f, e, 0x07060302u);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint32_t at = c0 + cq * 4 + k;
      if (at < p.cols) *reinterpret_cast<uint32_t*>(p.qt + at * p.ldqt + r0 + rq * 4) = o[k];
    }
  }
}

bool sizes_ok(int64_t batch, int64_t rows, int64_t cols) {
  constexpr int64_t most = (int64_t(1) << 31) - 256;
  if (batch < 0 || rows < 0 || cols < 0 || batch > most || rows > most || cols > most) return false;
  if (!batch || !rows || !cols) return true;
  const int64_t kb = (cols + 127) / 128;
  return batch * rows <= most && batch * rows <= most * 2 / kb;
}

int launch(void (*kernel)(QuantArgs), uint64_t groups, uint32_t threads, const QuantArgs& p, hipStream_t s) {
  MM_CHECK_ARG(groups * threads < uint64_t(1) << 32, "mm_quantize_blocks: too many blocks");  // what a grid holds
  kernel<<<static_cast<uint32_t>(groups), threads, 0, s>>>(p);
  return mm_check_launch("mm_quantize_blocks");
}

template <class T>
int launch_rows(const QuantArgs& p, hipStream_t s) {
  return launch(quantize_rows_kernel<T>, (p.units + 63) / 64, 256, p, s);
}

template <class T, bool BLOCK>
int launch_tiles(const QuantArgs& p, hipStream_t s) {
  const uint64_t tiles = static_cast<uint64_t>(p.batch) * ((p.rows + 127) / 128) * p.kb;
  // 1024 threads a tile wait for fewer loads each (1021 x 1793, 120 tiles: 4.8 us, 6.8 with 256; with a scale for
  // each row and column 6.0 and 9.5, and 28 and 30.5 for 2048 tiles); past two tiles a CU, 256 threads overlap more
  // tiles where one scale leaves little to compute (1024 tiles: 13.7 and 12.9)
  if constexpr (BLOCK) {
    if (tiles > 512) return launch(quantize_tile_kernel<T, BLOCK, 256>, tiles, 256, p, s);
  }
  return launch(quantize_tile_kernel<T, BLOCK, 1024>, tiles, 1024, p, s);
}

}  // namespace

extern "C" int mm_quantize_blocks(const void* x, int64_t ldx, int64_t x_batch, int32_t x_type, int64_t batch,
                                  int64_t rows, int64_t cols, int32_t block_rows, uint8_t* q, int64_t ldq,
                                  uint8_t* scale, mm_stream_t stream) {
  MM_CHECK_ARG(sizes_ok(batch, rows, cols), "mm_quantize_blocks: bad sizes (%lld x %lld x %lld)",
               static_cast<long long>(batch), static_cast<long long>(rows), static_cast<long long>(cols));
  MM_CHECK_ARG((x_type == MM_T_BF16 || x_type == MM_T_FP16 || x_type == MM_T_FP32) &&
                   (block_rows == 1 || block_rows == kBlock),
               "mm_quantize_blocks: bad type or block");
  const int64_t kb = (cols + 127) / 128;
  MM_CHECK_ARG(ldq >= cols && ldq <= kb * kBlock, "mm_quantize_blocks: rows of q must be %lld to %lld apart",
               static_cast<long long>(cols), static_cast<long long>(kb * kBlock));
  if (!batch || !rows || !cols) return MM_OK;
  MM_CHECK_ARG(x && q && scale, "mm_quantize_blocks: null pointer");
  const QuantArgs p{x, nullptr, q, scale, nullptr, nullptr, ldx, x_batch, ldq, 0, static_cast<uint32_t>(batch),
                    static_cast<uint32_t>(rows), static_cast<uint32_t>(cols), static_cast<uint32_t>(kb),
                    static_cast<uint64_t>(batch) * rows * kb};
  const hipStream_t s = mm_hip_stream(stream);
  if (block_rows == 1) {
    if (x_type == MM_T_FP32) return launch_rows<float>(p, s);
    return x_type == MM_T_FP16 ? launch_rows<_Float16>(p, s) : launch_rows<bf16>(p, s);
  }
  if (x_type == MM_T_FP32) return launch_tiles<float, true>(p, s);
  return x_type == MM_T_FP16 ? launch_tiles<_Float16, true>(p, s) : launch_tiles<bf16, true>(p, s);
}

extern "C" int mm_quantize_blocks_t(const void* x, int64_t ldx, int32_t x_type, const uint8_t* x_scale, int64_t rows,
                                    int64_t cols, int32_t block_rows, uint8_t* q, uint8_t* scale, uint8_t* qt,
                                    uint8_t* scale_t, mm_stream_t stream) {
  MM_CHECK_ARG(sizes_ok(1, rows, cols), "mm_quantize_blocks_t: bad sizes (%lld x %lld)", static_cast<long long>(rows),
               static_cast<long long>(cols));
  const bool eight = x_type == MM_T_E4M3;
  MM_CHECK_ARG((eight || x_type == MM_T_BF16 || x_type == MM_T_FP16 || x_type == MM_T_FP32) &&
                   (block_rows == 1 || block_rows == kBlock) && (!eight || (block_rows == kBlock && !q)),
               "mm_quantize_blocks_t: bad type or block");
  if (!rows || !cols) return MM_OK;
  MM_CHECK_ARG(x && qt && scale_t && (!q || scale) && (!eight || x_scale), "mm_quantize_blocks_t: null pointer");
  const int64_t kb = (cols + 127) / 128, rb = (rows + 127) / 128;
  const QuantArgs p{x, x_scale, q, scale, qt, scale_t, ldx, 0, kb * kBlock, rb * kBlock, 1, static_cast<uint32_t>(rows),
                    static_cast<uint32_t>(cols), static_cast<uint32_t>(kb), static_cast<uint64_t>(rows) * kb};
  const hipStream_t s = mm_hip_stream(stream);
  if (eight) return launch_tiles<E4m3, true>(p, s);
  if (block_rows == 1) {
    if (x_type == MM_T_FP32) return launch_tiles<float, false>(p, s);
    return x_type == MM_T_FP16 ? launch_tiles<_Float16, false>(p, s) : launch_tiles<bf16, false>(p, s);
  }
  if (x_type == MM_T_FP32) return launch_tiles<float, true>(p, s);
  return x_type == MM_T_FP16 ? launch_tiles<_Float16, true>(p, s) : launch_tiles<bf16, true>(p, s);
}
