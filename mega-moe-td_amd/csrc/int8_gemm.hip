// Product of 8-bit integer rows with scales for each token and each channel.
//
//   out[m, n] = sa[m] * sb[n] * sum_k a[m, k] * b[n, k]  (+ bias[n])
//
// a [M, K] and b [N, K] are int8 with K contiguous. The sum is exact in int32
// (|sum| <= 2^14 K < 2^31 for K < 2^17), the scales and the bias are applied
// in fp32 and the result is rounded once to the output's type.
#include <type_traits>

#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
// What results are stored in, at any alignment of their type. One value, not
// elements: the compiler breaks an array's copy up to share it with the branch
// for a row's end (4096 x 256 x 4096: 24 us, 18 so).
typedef int Out4 __attribute__((ext_vector_type(4), aligned(2)));
typedef int Out2 __attribute__((ext_vector_type(2), aligned(2)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kMaxK = (1 << 17) - 1;
constexpr int64_t kMaxStride = int64_t(1) << 23;  // 256 rows of a tile in 32-bit offsets
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

// Workgroup id -> tile: the ids of an XCD (congruent mod 8) take a run of tiles,
// 8 rows of tiles deep, so that rows and channels are reused from its L2.
__device__ __forceinline__ void tile_of(int num_m, int num_n, int& mt, int& nt) {
  const int total = num_m * num_n, per = total / 8, rest = total % 8, x = blockIdx.x & 7;
  const int l = x * per + min(x, rest) + (blockIdx.x >> 3);
  constexpr int DEEP = 8;
  const int group = l / (DEEP * num_n), first = group * DEEP, rows = min(DEEP, num_m - first), in = l - group * DEEP * num_n;
  mt = first + in % rows;
  nt = in / rows;
}

__device__ __forceinline__ float load_any(const void* p, int type, int64_t at) {
  if (type == MM_T_FP32) return static_cast<const float*>(p)[at];
  if (type == MM_T_FP16) return static_cast<float>(static_cast<const _Float16*>(p)[at]);
  return static_cast<float>(static_cast<const bf16*>(p)[at]);
}

// Four results in 16 bits each.
__device__ __forceinline__ uint2 pack4(const f32x4& f, int out_type) {
  return out_type == MM_T_FP16 ? make_uint2(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]))
                               : make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
}

// Columns col .. col + 3 of a row, from their sums.
__device__ __forceinline__ void store4(const I8Args& p, int row, int col, const i32x4& v) {
  const int left = p.n - col;
  const float sa = p.sa[row];
  f32x4 f;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int at = min(col + r, p.n - 1);
    f[r] = static_cast<float>(v[r]) * sa * p.sb[at] + (p.bias ? load_any(p.bias, p.bias_type, at) : 0.0f);
  }
  const int64_t at = row * p.ldo + col;
  if (p.out_type == MM_T_FP32) {
    float* out = static_cast<float*>(p.out) + at;
    if (left >= 4) {
      *reinterpret_cast<Out4*>(out) = __builtin_bit_cast(i32x4, f);
    } else {
#pragma unroll
      for (int r = 0; r < 3; ++r)
        if (r < left) out[r] = f[r];
    }
    return;
  }
  const uint2 h = pack4(f, p.out_type);
  uint16_t* out = static_cast<uint16_t*>(p.out) + at;
  if (left >= 4) {
    *reinterpret_cast<Out2*>(out) = Out2{static_cast<int>(h.x), static_cast<int>(h.y)};
  } else {
    if (left > 0) out[0] = static_cast<uint16_t>(h.x);
    if (left > 1) out[1] = static_cast<uint16_t>(h.x >> 16);
    if (left > 2) out[2] = static_cast<uint16_t>(h.y);
  }
}

// Sixteen bytes of a row as an operand. Rows that do not begin on 4-byte
// borders (SHIFT) are read as the five aligned words around them and shifted:
// 16-byte loads from odd addresses take the memory pipe twice as long (1021 x
// 2305 x 1793 in 64 x 64 tiles: 23 us that way, 21 this; 8 x 7169 x 4096: 23
// against 12). A word is read only if it holds a byte of the sixteen. `base` is
// aligned to 4 and the same for the wave.
__device__ __forceinline__ i32x4 join16(const uint32_t (&d)[5], uint32_t sh) {
  i32x4 v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = static_cast<int>(__builtin_amdgcn_alignbyte(d[i + 1], d[i], sh));
  return v;
}

template <bool SHIFT>
__device__ __forceinline__ i32x4 load16(const char* base, uint32_t off) {
  if constexpr (!SHIFT) {
    i32x4 v;
    __builtin_memcpy(&v, base + off, 16);
    return v;
  } else {
    const uint32_t sh = off & 3;
    const char* p = base + (off - sh);
    uint32_t d[5];
    __builtin_memcpy(d, __builtin_assume_aligned(p, 4), 16);
    __builtin_memcpy(d + 4, __builtin_assume_aligned(p + (sh ? 16 : 12), 4), 4);
    return join16(d, sh);
  }
}

// The same of a row with n bytes left: bytes past them read as zero and are
// not touched.
__device__ __forceinline__ i32x4 load16_cut(const char* base, uint32_t off, int n) {
  const int sh = off & 3;
  const uint32_t* p = reinterpret_cast<const uint32_t*>(base + (off - sh));
  uint32_t d[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) d[i] = n > 0 && 4 * i < n + sh && 4 * i < 16 + sh ? p[i] : 0;
  i32x4 v = join16(d, sh);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int keep = n - 4 * i;
    v[i] &= keep >= 4 ? -1 : keep <= 0 ? 0 : (1 << (8 * keep)) - 1;
  }
  return v;
}

// Address of a row as an aligned base and what is left of it.
__device__ __forceinline__ const char* aligned_base(const int8_t* p, uint32_t& rest) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  rest = a & 3;
  return reinterpret_cast<const char*>(a - rest);
}

// ------------------------------------------------------------------ operands from memory
// Tile of 16 G channels x 16 NT tokens for products that a grid of large tiles
// would not fill the chip with. Channels are the rows of v_mfma_i32_16x16x64_i8
// and tokens its columns; 16 bytes of a row are a lane's operand as they lie in
// memory. The W waves share the sum's axis in pieces of 128 bytes (wave w takes
// w, w + W, ...), U of them in flight, and join through LDS.
template <int G, int NT, int W, int U, bool SHIFT>
__global__ __launch_bounds__(W * 64) void int8_direct_kernel(I8Args p) {
  __shared__ i32x4 red[W * G * NT * 64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  // every XCD gets a run of channels with all their tokens
  const int total = gridDim.x, per = (total + 7) / 8, tiles_m = (p.m + NT * 16 - 1) / (NT * 16);
  int tile = blockIdx.x;
  if (total % 8 == 0) tile = (tile & 7) * per + (tile >> 3);
  const int n0 = tile / tiles_m * (G * 16), m0 = tile % tiles_m * (NT * 16);
  uint32_t b_off[G], a_off[NT], rest_a, rest_b;
  const char* a = aligned_base(p.a + m0 * p.lda, rest_a);
  const char* b = aligned_base(p.b + n0 * p.ldb, rest_b);
#pragma unroll
  for (int g = 0; g < G; ++g)
    b_off[g] = static_cast<uint32_t>(min(g * 16 + j, p.n - 1 - n0)) * static_cast<uint32_t>(p.ldb) + rest_b + 16 * q;
#pragma unroll
  for (int n = 0; n < NT; ++n)
    a_off[n] = static_cast<uint32_t>(min(n * 16 + j, p.m - 1 - m0)) * static_cast<uint32_t>(p.lda) + rest_a + 16 * q;
  i32x4 acc[G][NT];
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[g][n] = i32x4{0, 0, 0, 0};
  const int full = p.k / 128;
  auto steps = [&](auto count, int s) {
    constexpr int C = decltype(count)::value;
    i32x4 bv[C][G][2], av[C][NT][2];
#pragma unroll
    for (int u = 0; u < C; ++u) {
      const int at = (s + u * W) * 128;
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int h = 0; h < 2; ++h) bv[u][g][h] = load16<SHIFT>(b + at + h * 64, b_off[g]);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) av[u][n][h] = load16<SHIFT>(a + at + h * 64, a_off[n]);
    }
#pragma unroll
    for (int u = 0; u < C; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            acc[g][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bv[u][g][h], av[u][n][h], acc[g][n], 0, 0, 0);
  };
  int s = wave;
  for (; s + (U - 1) * W < full; s += U * W) steps(std::integral_constant<int, U>{}, s);
  for (; s < full; s += W) steps(std::integral_constant<int, 1>{}, s);
  if (p.k % 128 && s == full) {  // the last piece of the sum, cut at K
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = full * 128 + h * 64;
      i32x4 bv[G], av[NT];
#pragma unroll
      for (int g = 0; g < G; ++g) bv[g] = load16_cut(b + at, b_off[g], p.k - at - 16 * q);
#pragma unroll
      for (int n = 0; n < NT; ++n) av[n] = load16_cut(a + at, a_off[n], p.k - at - 16 * q);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[g][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(bv[g], av[n], acc[g][n], 0, 0, 0);
    }
  }
#pragma unroll
  for (int g = 0; g < G; ++g)
#pragma unroll
    for (int n = 0; n < NT; ++n) red[(wave * G * NT + n * G + g) * 64 + lane] = acc[g][n];
  __syncthreads();
  for (int op = wave; op < G * NT; op += W) {
    i32x4 v = red[op * 64 + lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += red[(w * G * NT + op) * 64 + lane];
    const int row = m0 + op / G * 16 + j;
    if (row < p.m) store4(p, row, n0 + op % G * 16 + 4 * q, v);
  }
}

// ------------------------------------------------------------------ tiles through LDS
// BM x BN tile, WM x WN waves of (BM / WM) x (BN / WN) in v_mfma_i32_32x32x32_i8
// blocks. Stages of 128 bytes of the sum's axis go through registers, PRE
// stages ahead, into a ring of two LDS buffers; one barrier a stage. The
// operands are swapped, so a lane holds 4 consecutive columns of one row.
//
// A sum in int32 has no order: the stage that K cuts comes first, with its
// missing bytes zeroed, and every other stage is whole.
//
// With KS > 1 a stage is KS pieces of 128 bytes, one for each of KS groups of
// WM x WN waves; the groups' sums are joined at the end. Products of few tiles
// then have KS times fewer stages, one after the other, and KS times the bytes
// in flight.
constexpr int BK = 128;

// LDS rows of 128 bytes: 16-byte slot s of row r sits at s ^ ((r >> 1) & 7),
// which gives the 16 rows of one pass of a fragment read distinct banks.
__device__ __forceinline__ int slot_of(int r, int s) { return r * BK + ((s ^ ((r >> 1) & 7)) << 4); }

// ROWS rows of a stage: KS sub-panels of [ROWS][128], filled by NT threads. With
// SHIFT a vector's fifth word is the first of the next lane's vector; only the
// last lane of a run loads it, and words are joined on their way to LDS (128 x
// 7169 x 4096 in 32 x 64 tiles: 21 us, 23 with five words loaded by every lane).
template <int ROWS, int NT, int KS, bool SHIFT>
struct Panel {
  static constexpr int VPR = 8 * KS, PER = ROWS * VPR / NT;  // 16-byte vectors a row, a thread
  static_assert(PER * NT == ROWS * VPR && NT % VPR == 0, "whole vectors");
  // A run: consecutive lanes with consecutive vectors of a row, within the 16
  // lanes that exchange words.
  static constexpr int LAST = VPR < 16 ? VPR - 1 : 15;
  struct Stage {
    uint32_t d[PER][SHIFT ? 5 : 4];
  };
  const char* base;
  uint32_t off[PER];
  __device__ __forceinline__ void init(const int8_t* p, int64_t ld, int r0, int rows) {
    uint32_t rest;
    base = aligned_base(p + r0 * ld, rest);
#pragma unroll
    for (int v = 0; v < PER; ++v) {
      const int c = v * NT + threadIdx.x;
      off[v] = static_cast<uint32_t>(min(c / VPR, rows - 1 - r0)) * static_cast<uint32_t>(ld) + rest + c % VPR * 16;
    }
  }
  __device__ __forceinline__ static bool last_of_run() { return (threadIdx.x & LAST) == LAST; }
  __device__ __forceinline__ void load(Stage& r, int k) const {
#pragma unroll
    for (int v = 0; v < PER; ++v) {
      if constexpr (SHIFT) {
        const uint32_t sh = off[v] & 3;
        const char* p = base + k + (off[v] - sh);
        __builtin_memcpy(r.d[v], __builtin_assume_aligned(p, 4), 16);
        if (last_of_run()) __builtin_memcpy(r.d[v] + 4, __builtin_assume_aligned(p + (sh ? 16 : 12), 4), 4);
      } else {
        __builtin_memcpy(r.d[v], base + k + off[v], 16);
      }
    }
  }
  __device__ __forceinline__ void put(int8_t* lds, const Stage& r) const {
#pragma unroll
    for (int v = 0; v < PER; ++v) {
      if constexpr (SHIFT) {
        uint32_t d[5];
#pragma unroll
        for (int i = 0; i < 5; ++i) d[i] = r.d[v][i];
        const uint32_t next = __builtin_amdgcn_update_dpp(d[4], d[0], 0x101, 0xf, 0xf, false);  // of lane + 1
        if (!last_of_run()) d[4] = next;
        put(lds, v, join16(d, off[v] & 3));
      } else {
        i32x4 x;
        __builtin_memcpy(&x, r.d[v], 16);
        put(lds, v, x);
      }
    }
  }
  // The stage that K cuts, from memory to LDS.
  __device__ __forceinline__ void put_cut(int8_t* lds, int k, int K) const {
    const int in = threadIdx.x % VPR * 16;  // the same for all of a thread's vectors
    i32x4 x[PER];
#pragma unroll
    for (int v = 0; v < PER; ++v) x[v] = load16_cut(base + k, off[v], K - k - in);
#pragma unroll
    for (int v = 0; v < PER; ++v) put(lds, v, x[v]);
  }
  __device__ __forceinline__ static void put(int8_t* lds, int v, const i32x4& x) {
    const int c = v * NT + threadIdx.x, s = c % VPR;
    *reinterpret_cast<i32x4*>(lds + s / 8 * ROWS * BK + slot_of(c / VPR, s % 8)) = x;
  }
};

// 32 staged rows of a wave to memory, 16 bytes a lane.
template <int COLS, int PITCH, class T>
__device__ __forceinline__ void store_rows(const I8Args& p, const int8_t* staged, int row0, int col0) {
  constexpr int PER = 16 / sizeof(T), LANES = COLS / PER;  // columns a lane, lanes a row
  const int lane = threadIdx.x & 63, r0 = lane / LANES, c = lane % LANES * PER, left = p.n - col0 - c;
  T* out = static_cast<T*>(p.out) + (row0 + r0) * p.ldo + col0 + c;
  const int64_t step = 64 / LANES * p.ldo;
#pragma unroll
  for (int r = 0; r < 32; r += 64 / LANES, out += step) {
    if (row0 + r0 + r >= p.m) break;
    const int8_t* from = staged + (r0 + r) * PITCH + c * sizeof(T);
    if (left >= PER) {
      *reinterpret_cast<Out4*>(out) = *reinterpret_cast<const i32x4*>(from);
    } else {
      for (int u = 0; u < left; ++u) out[u] = reinterpret_cast<const T*>(from)[u];
    }
  }
}

template <int BM, int BN, int WM, int WN, int KS, int PRE, bool SHIFT>
__global__ __launch_bounds__(WM * WN * KS * 64) void int8_tile_kernel(I8Args p) {
  constexpr int NT = WM * WN * KS * 64, STEP = KS * BK, MI = BM / WM / 32, NI = BN / WN / 32;
  __shared__ __attribute__((aligned(1024))) int8_t smem[2][(BM + BN) * STEP];
  const int num_m = (p.m + BM - 1) / BM, num_n = (p.n + BN - 1) / BN;
  int mt, nt;
  tile_of(num_m, num_n, mt, nt);
  const int m0 = mt * BM, n0 = nt * BN;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ks = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
  using PanelA = Panel<BM, NT, KS, SHIFT>;
  using PanelB = Panel<BN, NT, KS, SHIFT>;
  PanelA pa;
  PanelB pb;
  pa.init(p.a, p.lda, m0, p.m);
  pb.init(p.b, p.ldb, n0, p.n);
  // the tile's scales and bias, for the epilogue: a row and a channel a thread
  __shared__ __attribute__((aligned(16))) float row_scale[BM], col_scale[BN], col_bias[BN];
  static_assert(NT >= BM && NT >= BN, "a thread for each");
  if (threadIdx.x < BM) row_scale[threadIdx.x] = p.sa[min(m0 + static_cast<int>(threadIdx.x), p.m - 1)];
  if (threadIdx.x < BN) {
    const int channel = min(n0 + static_cast<int>(threadIdx.x), p.n - 1);
    col_scale[threadIdx.x] = p.sb[channel];
    col_bias[threadIdx.x] = p.bias ? load_any(p.bias, p.bias_type, channel) : 0.0f;
  }
  i32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0;

  const int cut = p.k % STEP, stages = (p.k + STEP - 1) / STEP;
  typename PanelA::Stage ra[PRE];
  typename PanelB::Stage rb[PRE];
  // stage s > 0 begins at byte (s - 1) * STEP, or s * STEP where K cuts none
  const int shift = cut ? STEP : 0;
  if (cut) {
    pa.put_cut(smem[0], p.k - cut, p.k);
    pb.put_cut(smem[0] + BM * STEP, p.k - cut, p.k);
  } else {
    pa.load(ra[0], 0);
    pb.load(rb[0], 0);
    pa.put(smem[0], ra[0]);
    pb.put(smem[0] + BM * STEP, rb[0]);
  }
  // loads past the last stage repeat it (K >= STEP: there is a whole one)
  auto at = [&](int s) { return max(min(s, stages - 1) * STEP - shift, 0); };
#pragma unroll
  for (int u = 0; u < PRE; ++u) {
    pa.load(ra[u], at(u + 1));
    pb.load(rb[u], at(u + 1));
  }
  __syncthreads();
  i32x4 fa[2][MI], fb[2][NI];
  auto frags = [&](int set, const int8_t* buf, int kk) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
      fa[set][i] = *reinterpret_cast<const i32x4*>(
          buf + ks * BM * BK + slot_of(wm * (BM / WM) + i * 32 + (lane & 31), kk * 2 + (lane >> 5)));
#pragma unroll
    for (int j = 0; j < NI; ++j)
      fb[set][j] = *reinterpret_cast<const i32x4*>(
          buf + BM * STEP + ks * BN * BK + slot_of(wn * (BN / WN) + j * 32 + (lane & 31), kk * 2 + (lane >> 5)));
  };
  auto mfmas = [&](int set) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NI; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(fb[set][j], fa[set][i], acc[i][j], 0, 0, 0);
  };
  frags(0, smem[0], 0);
  // Sub-steps of 32 bytes: the next one's fragments are read while this one
  // multiplies. Stage s + 1 goes from its registers to LDS in sub-steps 0 (a)
  // and 1 (b) and its registers take stage s + 1 + PRE; the barrier after
  // sub-step 2 publishes it, and its first fragments are read in sub-step 3.
  // Past the last stage the writes land where nobody reads any more.
  auto stage = [&](int s, auto reg) __attribute__((always_inline)) {
    constexpr int R = decltype(reg)::value;
    const int8_t* cur = smem[s & 1];
    int8_t* nxt = smem[(s + 1) & 1];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      frags((kk + 1) & 1, kk < 3 ? cur : nxt, (kk + 1) & 3);
      mfmas(kk & 1);
      if (kk == 0) {
        pa.put(nxt, ra[R]);
        pa.load(ra[R], at(s + 1 + PRE));
      }
      if (kk == 1) {
        pb.put(nxt + BM * STEP, rb[R]);
        pb.load(rb[R], at(s + 1 + PRE));
      }
#pragma unroll
      for (int g = 0; g < MI * NI; ++g) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // LDS read
        __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);  // LDS write
        __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // global load
      }
      if (kk == 2) __syncthreads();
    }
  };
  for (int s = 0; s < stages; s += PRE) {
    stage(s, std::integral_constant<int, 0>{});
    if constexpr (PRE > 1) {
      if (s + 1 < stages) stage(s + 1, std::integral_constant<int, 1>{});
    }
  }

  // Epilogue: sums are scaled and rounded where they lie (a lane has 4
  // consecutive columns of one row in each quarter of a block); 32 rows of a
  // wave at a time go through its own LDS, padded to spread a pass over the
  // banks, so that neighbouring lanes store neighbouring 16 bytes.
  constexpr int COLS = BN / WN, PITCH = COLS * 4 + 16, PITCH16 = COLS * 2 + 16;  // bytes of a staged row
  static_assert(WM * WN * 32 * PITCH <= sizeof(smem), "epilogue staging");
  __syncthreads();
  if constexpr (KS > 1) {  // group 0 adds the others' sums, one group at a time
    static_assert(BM * BN * 4 <= sizeof(smem), "a group's sums");
    i32x4* red = reinterpret_cast<i32x4*>(&smem[0][0]) + (wm * WN + wn) * (MI * NI * 4 * 64) + lane;
    for (int k = 1; k < KS; ++k) {
      if (ks == k) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g)
              red[((i * NI + j) * 4 + g) * 64] =
                  i32x4{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
      }
      __syncthreads();
      if (ks == 0) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
          for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const i32x4 v = red[((i * NI + j) * 4 + g) * 64];
#pragma unroll
              for (int r = 0; r < 4; ++r) acc[i][j][4 * g + r] += v[r];
            }
      }
      __syncthreads();
    }
    if (ks) return;
  }
  int8_t* const staged = &smem[0][0] + wave * (32 * PITCH);
  const int c0 = wn * COLS, lane_row = lane & 31, lane_col = lane >> 5 << 2;
  f32x4 sc[NI][4], bi[NI][4];
#pragma unroll
  for (int j = 0; j < NI; ++j)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = c0 + j * 32 + g * 8 + lane_col;
      sc[j][g] = *reinterpret_cast<const f32x4*>(col_scale + c);
      bi[j][g] = *reinterpret_cast<const f32x4*>(col_bias + c);
    }
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int r0 = wm * (BM / WM) + i * 32;
    const float s = row_scale[r0 + lane_row];
    // the lane's four results in quarter g of block j
    auto results = [&](int j, int g) __attribute__((always_inline)) {
      f32x4 f;
#pragma unroll
      for (int r = 0; r < 4; ++r) f[r] = static_cast<float>(acc[i][j][4 * g + r]) * s * sc[j][g][r] + bi[j][g][r];
      return f;
    };
    if (p.out_type == MM_T_FP32) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<f32x4*>(staged + lane_row * PITCH + (j * 32 + g * 8 + lane_col) * 4) = results(j, g);
      store_rows<COLS, PITCH, float>(p, staged, m0 + r0, n0 + c0);
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint2*>(staged + lane_row * PITCH16 + (j * 32 + g * 8 + lane_col) * 2) =
              pack4(results(j, g), p.out_type);
      store_rows<COLS, PITCH16, uint16_t>(p, staged, m0 + r0, n0 + c0);
    }
  }
}

// ------------------------------------------------------------------ choice
int launch(void (*kernel)(I8Args), int64_t tiles, int threads, const I8Args& p, hipStream_t s) {
  MM_CHECK_ARG(tiles * threads < (int64_t(1) << 32), "mm_int8_matmul: too many tiles");
  kernel<<<static_cast<uint32_t>(tiles), threads, 0, s>>>(p);
  return mm_check_launch("int8_matmul");
}

int64_t tiles_of(const I8Args& p, int bm, int bn) {
  return ((static_cast<int64_t>(p.m) + bm - 1) / bm) * ((static_cast<int64_t>(p.n) + bn - 1) / bn);
}

template <int G, int NT, int W, int U>
int launch_direct(const I8Args& p, bool shift, hipStream_t s) {
  return launch(shift ? int8_direct_kernel<G, NT, W, U, true> : int8_direct_kernel<G, NT, W, U, false>,
                tiles_of(p, NT * 16, G * 16), W * 64, p, s);
}

template <int BM, int BN, int WM, int WN, int KS, int PRE, bool SHIFT>
int launch_tiles(const I8Args& p, hipStream_t s) {
  return launch(int8_tile_kernel<BM, BN, WM, WN, KS, PRE, SHIFT>, tiles_of(p, BM, BN), WM * WN * KS * 64, p, s);
}

// Time of a product in us by its tiles: every 256 of them take `round` + `byte`
// a byte of K, as measured on full rounds (and about 4 us in all). Tiles below
// 64 x 64 gain from the bytes they have in flight while the chip is not full.
// 128 x 64 tiles fill a CU's LDS alone and are for one round (512 x 7168 x
// 4096: 27 us, in 64 x 64 33; 968 x 4992 x 6016, two: 64 us, in 128 x 128 48).
struct TileCost {
  int bm, bn, step;  // step: K has to reach one whole stage
  double round, byte;
  int rounds = 1 << 30;  // for so many
};
constexpr TileCost kTileCosts[] = {
    {256, 256, 128, 11.5, 13.3e-3}, {128, 128, 128, 3.3, 5.0e-3}, {128, 64, 256, 4.0, 2.9e-3, 1},
    {64, 64, 128, 1.4, 1.75e-3},    {32, 64, 512, 1.8, 1.4e-3},   {32, 32, 1024, 1.8, 1.15e-3},
};

int best_tile(const I8Args& p) {
  int best = 0;
  double least = 1e300;
  for (int i = 0; i < 6; ++i) {
    const TileCost& c = kTileCosts[i];
    const int64_t rounds = (tiles_of(p, c.bm, c.bn) + 255) / 256;
    const double t = static_cast<double>(rounds) * (c.round + c.byte * p.k);
    if (p.k >= c.step && rounds <= c.rounds && t < least) best = i, least = t;
  }
  return best;
}

int launch_best(const I8Args& p, hipStream_t s) {
  // rows on 4-byte borders need no shifting; the two largest tiles leave odd
  // addresses to the memory pipe, which their longer stages hide (2048 x 4097 x
  // 4096: 80 us in 128 x 128 tiles against 90 with shifts)
  const bool shift = ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b) | p.lda | p.ldb) & 3) != 0;
  // 16 rows: 7168 x 4096 in 8 us, the smallest tiles 11
  if (p.m <= 16) return launch_direct<1, 1, 16, 4>(p, shift, s);
  if (p.k < BK) return launch_direct<4, 4, 1, 1>(p, shift, s);  // not one whole stage
  switch (best_tile(p)) {
    case 0: return launch_tiles<256, 256, 2, 2, 1, 1, false>(p, s);
    case 1: return launch_tiles<128, 128, 2, 2, 1, 2, false>(p, s);
    case 2:
      return shift ? launch_tiles<128, 64, 2, 2, 2, 2, true>(p, s) : launch_tiles<128, 64, 2, 2, 2, 2, false>(p, s);
    case 3:
      // the sum shared by two groups of waves until the chip is full (256 x
      // 7168 x 4096, 256 tiles: 18 us against 24; 464 tiles of 2309: 22 against 19)
      if (p.k >= 2 * BK && tiles_of(p, 64, 64) <= 256)
        return shift ? launch_tiles<64, 64, 2, 2, 2, 2, true>(p, s) : launch_tiles<64, 64, 2, 2, 2, 2, false>(p, s);
      return shift ? launch_tiles<64, 64, 2, 2, 1, 2, true>(p, s) : launch_tiles<64, 64, 2, 2, 1, 2, false>(p, s);
    case 4: return shift ? launch_tiles<32, 64, 1, 2, 4, 2, true>(p, s) : launch_tiles<32, 64, 1, 2, 4, 2, false>(p, s);
    default: return shift ? launch_tiles<32, 32, 1, 1, 8, 1, true>(p, s) : launch_tiles<32, 32, 1, 1, 8, 1, false>(p, s);
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
  MM_CHECK_ARG((m <= 1 || (lda >= k && lda <= kMaxStride)) && (n <= 1 || (ldb >= k && ldb <= kMaxStride)) &&
                   (m <= 1 || ldo >= n),
               "mm_int8_matmul: bad strides (rows of a and b at least K and at most %lld apart)",
               static_cast<long long>(kMaxStride));
  if (m == 0) return MM_OK;
  MM_CHECK_ARG(a && b && a_scale && b_scale && out, "mm_int8_matmul: null pointer");
  // a single row's stride is never stepped over
  if (m == 1) lda = k;
  if (n == 1) ldb = k;
  const I8Args p{a, b, a_scale, b_scale, bias, out, lda, ldb, ldo, static_cast<int32_t>(m), static_cast<int32_t>(n),
                 static_cast<int32_t>(k), out_type, bias_type};
  return launch_best(p, mm_hip_stream(stream));
}
