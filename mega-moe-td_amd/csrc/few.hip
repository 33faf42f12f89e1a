// The whole layer for a few tokens in two launches.
//
//   act[r, :] = act_fn(x[t] W1[e] gate, up) * w[r]      (r = t * k + j, e = selected[r])
//   out[t, :] = sum_j act[t * k + j, :] W2[e]^T
//
// A few tokens are bound by reading the weights of the experts they reach, and
// at one token by the launches in between. Here no routing tables exist: a
// workgroup owns (expert, columns), finds the expert's routes in `selected` by
// itself, and reads its weights once, straight into matrix-instruction
// operands. Weights are the instruction's rows and tokens its 16 columns, so 1
// to 16 rows of an expert cost the same and absent ones need no masking: a
// result column depends on its own token only. The 8 waves of a workgroup
// share the sum's axis and join through LDS in wave order. The second launch
// leaves fp32 rows in scratch; the workgroup that finishes a range of columns
// last adds the tokens' slots in slot order. Every sum has a fixed order.
#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 512, kWaves = 8;
constexpr int kMaxRoutes = 4096;  // 64 tokens of 64 slots
constexpr int kGroup = MM_FEW_ACT_GROUP;
constexpr float kScaleFloor = 1e-30f;

struct FewArgs {
  const void* x;              // [T, H] bf16 or int8
  const float* x_scale;       // [T], int8
  const int32_t* selected;    // [R]
  const float* w;             // [R]
  const void* w1;             // bf16 [E, H, 2I] or int8 [E, 2I, H]
  const float* w1_scale;      // [E, 2I], int8
  const void* w2;             // bf16, either unit stride, or int8 [E, H, I]
  const float* w2_scale;      // [E, H], int8
  int64_t w2_se, w2_ld;       // expert stride; stride of the axis that is not contiguous
  int32_t R, top_k, E, H, I, tokens, act_kind;
  float beta, lbeta, limit;
  void* act;                  // [R, I] bf16 or int8
  float* act_scale;           // [R, I / 32], int8
  float* y;                   // [R, H]
  int32_t* done;              // [column tiles + 1]: arrivals, then the number of distinct experts
  bf16* out;                  // [T, H]
  int32_t tiles, fc2_tiles;   // column tiles of this launch, and of the second
};

// A slot of the grid is an expert where the experts are no more than the
// routes, else a route, of which the first with its expert does the work.
// Fills `list` with the routes of the slot's expert in ascending order and
// returns their number, 0 if the slot has no work. Every wave scans for itself
// and writes the same values: no barrier.
__device__ __forceinline__ int find_routes(const FewArgs& p, int slot, uint16_t* list, int& expert) {
  const int lane = threadIdx.x & 63;
  const bool by_expert = p.E <= p.R;
  const int e = by_expert ? slot : __builtin_amdgcn_readfirstlane(p.selected[slot]);
  expert = e;
  if (static_cast<uint32_t>(e) >= static_cast<uint32_t>(p.E)) return 0;
  int count = 0;
  for (int base = 0; base < p.R; base += 64) {
    const int r = base + lane;
    const bool hit = r < p.R && p.selected[r] == e;
    const uint64_t mask = __ballot(hit);
    if (!by_expert && count == 0 && mask && base + __ffsll(static_cast<unsigned long long>(mask)) - 1 != slot) return 0;
    if (hit) list[count + __popcll(mask & ((1ull << lane) - 1))] = static_cast<uint16_t>(r);
    count += __popcll(mask);
  }
  return count;
}

// Clears the second launch's arrival counters and counts the distinct experts,
// each of which arrives once at every range of columns.
__device__ void prepare_done(const FewArgs& p, uint32_t* bits) {
  for (int i = threadIdx.x; i < p.fc2_tiles; i += kThreads) p.done[i] = 0;
  const int words = (p.E + 31) / 32;
  for (int i = threadIdx.x; i < words; i += kThreads) bits[i] = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < p.R; r += kThreads) {
    const uint32_t e = static_cast<uint32_t>(p.selected[r]);
    if (e < static_cast<uint32_t>(p.E)) atomicOr(&bits[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    int n = 0;
    for (int i = threadIdx.x; i < words; i += 64) n += __popc(bits[i]);
    for (int m = 32; m > 0; m >>= 1) n += __shfl_xor(n, m);
    if (threadIdx.x == 0) p.done[p.fc2_tiles] = n;
  }
  __syncthreads();
}

// ------------------------------------------------------------------ products
// Weights with their columns contiguous, CL columns a lane: 8 rows of CL
// columns are transposed in registers (4 v_perm for each 16 bytes) into CL
// operands of 16 columns x 32 rows. Column of operand c, row i: CL * i + c.
template <int CL>
struct ColumnWeights {
  static constexpr int DW = CL / 2;
  uint32_t raw[8][DW];
  __device__ __forceinline__ void load(const bf16* p, int64_t ld) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if constexpr (CL == 8) {
        const uint4 v = load_stream16(p + r * ld);
        raw[r][0] = v.x, raw[r][1] = v.y, raw[r][2] = v.z, raw[r][3] = v.w;
      } else {
        const uint2 v = load_stream8(p + r * ld);
        raw[r][0] = v.x, raw[r][1] = v.y;
      }
    }
  }
  __device__ __forceinline__ bf16x8 operand(int c) const {
    const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
    u32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_perm(raw[2 * i + 1][c >> 1], raw[2 * i][c >> 1], sel);
    return __builtin_bit_cast(bf16x8, v);
  }
};

// acc[c][n] += W^T x over this wave's steps of 32 rows (wave, wave + 8, ...).
// w: the lane's columns in row 8 * (lane / 16); x[n]: its token's values there.
template <int CL, int NT>
__device__ __forceinline__ void columns_product(f32x4 (&acc)[CL][NT], const bf16* w, int64_t ld,
                                                const bf16* const (&x)[NT], int steps, int wave) {
  ColumnWeights<CL> cw[2];
  bf16x8 xv[2][NT];
  auto load = [&](int buf, int s) {
    cw[buf].load(w + static_cast<int64_t>(s) * 32 * ld, ld);
#pragma unroll
    for (int n = 0; n < NT; ++n) __builtin_memcpy(&xv[buf][n], x[n] + s * 32, 16);
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int c = 0; c < CL; ++c) {
      const bf16x8 a = cw[buf].operand(c);
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[c][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, xv[buf][n], acc[c][n], 0, 0, 0);
    }
  };
  if (wave >= steps) return;
  load(0, wave);
  for (int s = wave; s < steps; s += 2 * kWaves) {
    if (s + kWaves < steps) load(1, s + kWaves);
    multiply(0);
    if (s + kWaves >= steps) break;
    if (s + 2 * kWaves < steps) load(0, s + 2 * kWaves);
    multiply(1);
  }
}

// Weights with the sum's axis contiguous: 16 bytes a lane are an operand as
// they are. G groups of 16 rows; steps of 64 elements take two instructions,
// so that both halves of a 128-byte line are asked for together.
template <int G, int NT>
__device__ __forceinline__ void rows_product(f32x4 (&acc)[G][NT], const bf16* w, int64_t ld,
                                             const bf16* const (&x)[NT], int steps, int wave) {
  bf16x8 wv[2][2][G], xv[2][2][NT];
  auto load = [&](int buf, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int g = 0; g < G; ++g)
        wv[buf][h][g] = __builtin_bit_cast(bf16x8, load_stream16(w + g * 16 * ld + s * 64 + h * 32));
#pragma unroll
      for (int n = 0; n < NT; ++n) __builtin_memcpy(&xv[buf][h][n], x[n] + s * 64 + h * 32, 16);
    }
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int n = 0; n < NT; ++n)
          acc[g][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv[buf][h][g], xv[buf][h][n], acc[g][n], 0, 0, 0);
  };
  if (wave >= steps) return;
  load(0, wave);
  for (int s = wave; s < steps; s += 2 * kWaves) {
    if (s + kWaves < steps) load(1, s + kWaves);
    multiply(0);
    if (s + kWaves >= steps) break;
    if (s + 2 * kWaves < steps) load(0, s + 2 * kWaves);
    multiply(1);
  }
}

// The same on int8 (steps of 128 bytes, instructions of 64). w[g]: the lane's
// row of group g at byte 16 * (lane / 16).
template <int G, int NT>
struct Int8Step {
  i32x4 w[2][G], x[2][NT];
  __device__ __forceinline__ void load(const int8_t* const (&wp)[G], const int8_t* const (&xp)[NT], int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int g = 0; g < G; ++g) w[h][g] = __builtin_bit_cast(i32x4, load_stream16(wp[g] + s * 128 + h * 64));
#pragma unroll
      for (int n = 0; n < NT; ++n) __builtin_memcpy(&x[h][n], xp[n] + s * 128 + h * 64, 16);
    }
  }
};

// Sums of the waves' partial results in wave order; item = operand * 64 + lane.
template <int N, class V>
__device__ __forceinline__ void leave_partials(V* red, const V* acc, int wave, int lane) {
#pragma unroll
  for (int i = 0; i < N; ++i) red[(wave * N + i) * 64 + lane] = acc[i];
}
template <int N, class V>
__device__ __forceinline__ V join_partials(const V* red, int item) {
  V s = red[item];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) s += red[w * N * 64 + item];
  return s;
}

// ------------------------------------------------------------------ first launch, bf16
// Tile of C = 8 * CL columns: operand rows 0..7 are gate, 8..15 up columns.
template <int CL, int NT>
__global__ __launch_bounds__(kThreads) void few_fc1_kernel(FewArgs p) {
  constexpr int C = 8 * CL;
  __shared__ f32x4 red[kWaves * CL * NT * 64];
  __shared__ uint16_t list[kMaxRoutes];
  __shared__ __attribute__((aligned(16))) bf16 stage[NT * 16][C + 8];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, q = lane >> 4;
  if (blockIdx.x == 0) prepare_done(p, reinterpret_cast<uint32_t*>(red));
  const int slot = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  int e;
  const int count = find_routes(p, slot, list, e);
  if (!count) return;
  const int64_t ld = 2 * static_cast<int64_t>(p.I);
  const bf16* w = static_cast<const bf16*>(p.w1) + static_cast<int64_t>(e) * p.H * ld + static_cast<int64_t>(8 * q) * ld +
                  (j < 8 ? 0 : p.I) + tile * C + CL * (j & 7);
  for (int c0 = 0; c0 < count; c0 += 16 * NT) {
    const bf16* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      x[n] = static_cast<const bf16*>(p.x) +
             static_cast<int64_t>(list[min(c0 + n * 16 + j, count - 1)] / p.top_k) * p.H + 8 * q;
    f32x4 acc[CL][NT];
#pragma unroll
    for (int c = 0; c < CL; ++c)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[c][n] = f32x4{0, 0, 0, 0};
    columns_product<CL, NT>(acc, w, ld, x, p.H / 32, wave);
    leave_partials<CL * NT>(red, &acc[0][0], wave, lane);
    __syncthreads();
    for (int item = tid; item < CL * NT * 64; item += kThreads) {
      const int c = (item >> 6) / NT, n = (item >> 6) % NT;
      const f32x4 v = join_partials<CL * NT>(red, item);
      const int at = c0 + n * 16 + j;
      const float wt = p.w[list[min(at, count - 1)]];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float up = __shfl(v[r], (lane + 32) & 63);
        if (lane < 32)
          stage[n * 16 + j][CL * (4 * q + r) + c] =
              static_cast<bf16>(gated_act(p.act_kind, v[r], up, p.beta, p.lbeta, p.limit) * wt);
      }
    }
    __syncthreads();
    for (int item = tid; item < NT * 16 * (C / 8); item += kThreads) {
      const int row = item / (C / 8), vec = item % (C / 8);
      if (c0 + row < count)
        *reinterpret_cast<uint4*>(static_cast<bf16*>(p.act) + static_cast<int64_t>(list[c0 + row]) * p.I + tile * C +
                                  vec * 8) = *reinterpret_cast<const uint4*>(&stage[row][vec * 8]);
    }
  }
}

// ------------------------------------------------------------------ second launch
// Called by every workgroup with work once its part of y is written; the last
// of its range of columns adds the slots. C columns, column c of a row at
// place(c) of the range.
template <int C, class Place>
__device__ __forceinline__ void finish(const FewArgs& p, int tile, int live, Place place) {
  __shared__ int last;
  __threadfence();  // y of every thread is out before the workgroup arrives
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&p.done[tile], 1) == live - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();  // and the other workgroups' y is read behind their arrivals
  for (int i = threadIdx.x; i < p.tokens * C; i += kThreads) {
    const int t = i / C, c = i % C;
    const float* y = p.y + static_cast<int64_t>(t) * p.top_k * p.H + tile * C + place(c);
    float s = 0.0f;
    for (int k0 = 0; k0 < p.top_k; k0 += 8) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool in = k0 + k < p.top_k &&
                        static_cast<uint32_t>(p.selected[t * p.top_k + k0 + k]) < static_cast<uint32_t>(p.E);
        v[k] = in ? y[static_cast<int64_t>(k0 + k) * p.H] : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
    p.out[static_cast<int64_t>(t) * p.H + tile * C + c] = static_cast<bf16>(s);
  }
}

// No route has an expert: the first slot's workgroups write the empty sums.
template <int C>
__device__ __forceinline__ void finish_empty(const FewArgs& p, int tile) {
  for (int i = threadIdx.x; i < p.tokens * C; i += kThreads)
    p.out[static_cast<int64_t>(i / C) * p.H + tile * C + i % C] = static_cast<bf16>(0.0f);
}

// ROWS: w2's sum axis is contiguous (N = 4 groups of 16 columns), else its
// columns are (N = CL columns a lane).
template <bool ROWS, int N, int NT>
__global__ __launch_bounds__(kThreads) void few_fc2_kernel(FewArgs p) {
  constexpr int C = 16 * N;
  __shared__ f32x4 red[kWaves * N * NT * 64];
  __shared__ uint16_t list[kMaxRoutes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, q = lane >> 4;
  const int slot = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  const int live = p.done[p.tiles];
  if (live == 0 && slot == 0) finish_empty<C>(p, tile);
  int e;
  const int count = find_routes(p, slot, list, e);
  if (!count) return;
  const bf16* w = static_cast<const bf16*>(p.w2) + static_cast<int64_t>(e) * p.w2_se +
                  (ROWS ? static_cast<int64_t>(tile * C + j) * p.w2_ld + 8 * q
                        : static_cast<int64_t>(8 * q) * p.w2_ld + tile * C + N * j);
  for (int c0 = 0; c0 < count; c0 += 16 * NT) {
    const bf16* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      x[n] = static_cast<const bf16*>(p.act) + static_cast<int64_t>(list[min(c0 + n * 16 + j, count - 1)]) * p.I + 8 * q;
    f32x4 acc[N][NT];
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[c][n] = f32x4{0, 0, 0, 0};
    if constexpr (ROWS)
      rows_product<N, NT>(acc, w, p.w2_ld, x, p.I / 64, wave);
    else
      columns_product<N, NT>(acc, w, p.w2_ld, x, p.I / 32, wave);
    if (c0) __syncthreads();
    leave_partials<N * NT>(red, &acc[0][0], wave, lane);
    __syncthreads();
    // operand c, rows 4q..4q + 3 of token j are kept side by side in y
    for (int item = tid; item < N * NT * 64; item += kThreads) {
      const int c = (item >> 6) / NT, n = (item >> 6) % NT, at = c0 + n * 16 + j;
      const f32x4 v = join_partials<N * NT>(red, item);
      if (at < count)
        *reinterpret_cast<f32x4*>(p.y + static_cast<int64_t>(list[at]) * p.H + tile * C + c * 16 + 4 * q) = v;
    }
  }
  finish<C>(p, tile, live, [](int c) { return ROWS ? c : (c % N) * 16 + c / N; });
}

// ------------------------------------------------------------------ int8
// Tile of 32 columns: operands 0, 1 are gate columns, 2, 3 up columns.
template <int NT>
__global__ __launch_bounds__(kThreads) void few_fc1_int8_kernel(FewArgs p) {
  constexpr int C = kGroup, G = 4;
  __shared__ i32x4 red[kWaves * G * NT * 64];
  __shared__ uint16_t list[kMaxRoutes];
  __shared__ float stage[NT * 16][C + 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, q = lane >> 4;
  if (blockIdx.x == 0) prepare_done(p, reinterpret_cast<uint32_t*>(red));
  const int slot = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  int e;
  const int count = find_routes(p, slot, list, e);
  if (!count) return;
  const int8_t* w[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    w[g] = static_cast<const int8_t*>(p.w1) +
           (static_cast<int64_t>(e) * 2 * p.I + (g >> 1) * p.I + tile * C + (g & 1) * 16 + j) * p.H + 16 * q;
  const int steps = p.H / 128;
  for (int c0 = 0; c0 < count; c0 += 16 * NT) {
    const int8_t* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      x[n] = static_cast<const int8_t*>(p.x) +
             static_cast<int64_t>(list[min(c0 + n * 16 + j, count - 1)] / p.top_k) * p.H + 16 * q;
    i32x4 acc[G][NT];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[g][n] = i32x4{0, 0, 0, 0};
    Int8Step<G, NT> st[2];
    auto multiply = [&](const Int8Step<G, NT>& s) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int n = 0; n < NT; ++n) acc[g][n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.w[h][g], s.x[h][n], acc[g][n], 0, 0, 0);
    };
    if (wave < steps) {
      st[0].load(w, x, wave);
      for (int s = wave; s < steps; s += 2 * kWaves) {
        if (s + kWaves < steps) st[1].load(w, x, s + kWaves);
        multiply(st[0]);
        if (s + kWaves >= steps) break;
        if (s + 2 * kWaves < steps) st[0].load(w, x, s + 2 * kWaves);
        multiply(st[1]);
      }
    }
    leave_partials<G * NT>(red, &acc[0][0], wave, lane);
    __syncthreads();
    for (int item = tid; item < 2 * NT * 64; item += kThreads) {
      const int g = (item >> 6) / NT, n = (item >> 6) % NT;
      const i32x4 gate = join_partials<G * NT>(red, (g * NT + n) * 64 + lane);
      const i32x4 up = join_partials<G * NT>(red, ((g + 2) * NT + n) * 64 + lane);
      const int route = list[min(c0 + n * 16 + j, count - 1)];
      const float sx = p.x_scale[route / p.top_k], wt = p.w[route];
      const float* ws = p.w1_scale + static_cast<int64_t>(e) * 2 * p.I + tile * C + g * 16 + 4 * q;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        stage[n * 16 + j][g * 16 + 4 * q + r] =
            gated_act(p.act_kind, static_cast<float>(gate[r]) * (sx * ws[r]),
                      static_cast<float>(up[r]) * (sx * ws[p.I + r]), p.beta, p.lbeta, p.limit) * wt;
    }
    __syncthreads();
    // 32 lanes a row: its largest value (of the bit patterns, so that NaN shows), scale and bytes
    for (int item = tid; item < NT * 16 * C; item += kThreads) {
      const int row = item / C, col = item % C;
      const float v = stage[row][col];
      uint32_t top = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
      for (int m = 16; m > 0; m >>= 1) top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), m)));
      if (c0 + row >= count) continue;
      const bool finite = top < 0x7f800000u;
      const float a = fmaxf(__uint_as_float(top), kScaleFloor);
      const int route = list[c0 + row];
      static_cast<int8_t*>(p.act)[static_cast<int64_t>(route) * p.I + tile * C + col] =
          finite ? static_cast<int8_t>(static_cast<int>(__builtin_rintf(v * (127.0f / a)))) : 0;
      if (col == 0)
        p.act_scale[static_cast<int64_t>(route) * (p.I / C) + tile] = finite ? a / 127.0f : __uint_as_float(0x7fc00000u);
    }
  }
}

// Tile of 64 columns. An instruction's 64 elements span two scale groups (the
// operand's lanes 0..31 and 32..63), so each group is multiplied with the
// other's activations zeroed and joins the fp32 sum under its own scale.
template <int NT>
__global__ __launch_bounds__(kThreads) void few_fc2_int8_kernel(FewArgs p) {
  constexpr int G = 4, C = 16 * G;
  __shared__ f32x4 red[kWaves * G * NT * 64];
  __shared__ uint16_t list[kMaxRoutes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int j = lane & 15, q = lane >> 4;
  const int slot = blockIdx.x / p.tiles, tile = blockIdx.x % p.tiles;
  const int live = p.done[p.tiles];
  if (live == 0 && slot == 0) finish_empty<C>(p, tile);
  int e;
  const int count = find_routes(p, slot, list, e);
  if (!count) return;
  const int8_t* w[G];
#pragma unroll
  for (int g = 0; g < G; ++g)
    w[g] = static_cast<const int8_t*>(p.w2) + (static_cast<int64_t>(e) * p.H + tile * C + g * 16 + j) * p.I + 16 * q;
  const int steps = p.I / 128, groups = p.I / kGroup;
  for (int c0 = 0; c0 < count; c0 += 16 * NT) {
    const int8_t* x[NT];
    const float* sc[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int64_t route = list[min(c0 + n * 16 + j, count - 1)];
      x[n] = static_cast<const int8_t*>(p.act) + route * p.I + 16 * q;
      sc[n] = p.act_scale + route * groups;
    }
    f32x4 acc[G][NT];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[g][n] = f32x4{0, 0, 0, 0};
    Int8Step<G, NT> st[2];
    float sv[2][NT][4];
    auto load = [&](int buf, int s) {
      st[buf].load(w, x, s);
#pragma unroll
      for (int n = 0; n < NT; ++n) __builtin_memcpy(sv[buf][n], sc[n] + s * 4, 16);
    };
    auto multiply = [&](int buf) {
      const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const i32x4 lo = lane < 32 ? st[buf].x[h][n] : zero, hi = lane < 32 ? zero : st[buf].x[h][n];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const i32x4 a = __builtin_amdgcn_mfma_i32_16x16x64_i8(st[buf].w[h][g], lo, zero, 0, 0, 0);
            const i32x4 b = __builtin_amdgcn_mfma_i32_16x16x64_i8(st[buf].w[h][g], hi, zero, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[g][n][r] += static_cast<float>(a[r]) * sv[buf][n][2 * h] + static_cast<float>(b[r]) * sv[buf][n][2 * h + 1];
          }
        }
    };
    if (wave < steps) {
      load(0, wave);
      for (int s = wave; s < steps; s += 2 * kWaves) {
        if (s + kWaves < steps) load(1, s + kWaves);
        multiply(0);
        if (s + kWaves >= steps) break;
        if (s + 2 * kWaves < steps) load(0, s + 2 * kWaves);
        multiply(1);
      }
    }
    if (c0) __syncthreads();
    leave_partials<G * NT>(red, &acc[0][0], wave, lane);
    __syncthreads();
    for (int item = tid; item < G * NT * 64; item += kThreads) {
      const int g = (item >> 6) / NT, n = (item >> 6) % NT, at = c0 + n * 16 + j;
      f32x4 v = join_partials<G * NT>(red, item);
      const float* ws = p.w2_scale + static_cast<int64_t>(e) * p.H + tile * C + g * 16 + 4 * q;
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] *= ws[r];
      if (at < count)
        *reinterpret_cast<f32x4*>(p.y + static_cast<int64_t>(list[at]) * p.H + tile * C + g * 16 + 4 * q) = v;
    }
  }
  finish<C>(p, tile, live, [](int c) { return c; });
}

// ------------------------------------------------------------------ host
struct FewScratch {
  size_t act, act_scale, y, done, bytes;
  FewScratch(int64_t R, int64_t H, int64_t I, bool int8) {
    size_t at = 0;
    auto take = [&](size_t n) {
      const size_t p = at;
      at += mm_align_up(n, 256);
      return p;
    };
    act = take(static_cast<size_t>(R) * I * (int8 ? 1 : 2));
    act_scale = take(int8 ? static_cast<size_t>(R) * (I / kGroup) * 4 : 0);
    y = take(static_cast<size_t>(R) * H * 4);
    done = take((static_cast<size_t>(H) / 64 + 1) * 4);
    bytes = at;
  }
};

bool few_sizes_ok(int64_t tokens, int32_t top_k, int32_t E, int32_t H, int32_t I) {
  return tokens >= 0 && tokens <= MM_FEW_MAX_TOKENS && top_k > 0 && top_k <= 64 && E > 0 && E <= 32768 && H > 0 &&
         H % 128 == 0 && I > 0 && I % 128 == 0 && H <= (1 << 20) && I <= (1 << 20);
}

int slots_of(const FewArgs& p) { return p.E <= p.R ? p.E : p.R; }

// Two launches of (slots x column tiles) workgroups each.
template <class K1, class K2>
int launch_both(FewArgs p, int c1, K1 k1, int c2, K2 k2, hipStream_t s) {
  const int slots = slots_of(p), tiles1 = p.I / c1, tiles2 = p.H / c2;
  MM_CHECK_ARG(static_cast<int64_t>(slots) * (tiles1 > tiles2 ? tiles1 : tiles2) < (int64_t(1) << 23),
               "mm_moe_few: too many tiles");
  p.fc2_tiles = tiles2;
  p.tiles = tiles1;
  k1<<<slots * tiles1, kThreads, 0, s>>>(p);
  const int rc = mm_check_launch("few_fc1_kernel");
  if (rc) return rc;
  p.tiles = tiles2;
  k2<<<slots * tiles2, kThreads, 0, s>>>(p);
  return mm_check_launch("few_fc2_kernel");
}

}  // namespace

extern "C" size_t mm_moe_few_scratch_bytes(int64_t tokens, int32_t top_k, int32_t hidden, int32_t inter, int32_t int8) {
  if (!few_sizes_ok(tokens, top_k, 1, hidden, inter)) return 0;
  return FewScratch(tokens * top_k, hidden, inter, int8 != 0).bytes;
}

extern "C" int mm_moe_few(const uint16_t* x, const int32_t* selected, const float* routing_weights, const uint16_t* w1,
                          const uint16_t* w2, int64_t w2_se, int64_t w2_sh, int64_t w2_sf, int64_t tokens,
                          int32_t top_k, int32_t num_experts, int32_t hidden, int32_t inter, int32_t act_kind,
                          float situ_beta, float situ_linear_beta, float clamp_limit, uint16_t* out, void* scratch,
                          size_t scratch_bytes, mm_stream_t stream) {
  MM_CHECK_ARG(few_sizes_ok(tokens, top_k, num_experts, hidden, inter), "mm_moe_few: bad sizes");
  MM_CHECK_ARG(w2_sh == 1 || w2_sf == 1, "mm_moe_few: w2 needs a unit stride along hidden or inter");
  MM_CHECK_ARG(act_kind >= MM_ACT_SWIGLU && act_kind <= MM_ACT_CLAMP_SWIGLU, "mm_moe_few: bad activation");
  if (tokens == 0) return MM_OK;
  const FewScratch f(tokens * top_k, hidden, inter, false);
  MM_CHECK_ARG(x && selected && routing_weights && w1 && w2 && out && scratch, "mm_moe_few: null pointer");
  if (scratch_bytes < f.bytes) {
    mm_set_error("mm_moe_few: scratch needs %zu bytes", f.bytes);
    return MM_E_WS;
  }
  char* base = static_cast<char*>(scratch);
  const bool rows = w2_sf == 1;
  FewArgs p{x,      nullptr, selected, routing_weights, w1, nullptr, w2, nullptr, w2_se, rows ? w2_sh : w2_sf,
            static_cast<int32_t>(tokens * top_k), top_k, num_experts, hidden, inter, static_cast<int32_t>(tokens),
            act_kind, situ_beta, situ_linear_beta, clamp_limit, base + f.act, nullptr,
            reinterpret_cast<float*>(base + f.y), reinterpret_cast<int32_t*>(base + f.done),
            reinterpret_cast<bf16*>(out), 0, 0};
  const hipStream_t s = mm_hip_stream(stream);
  if (tokens <= 16) {
    if (rows) return launch_both(p, 32, few_fc1_kernel<4, 1>, 64, few_fc2_kernel<true, 4, 1>, s);
    return launch_both(p, 32, few_fc1_kernel<4, 1>, 64, few_fc2_kernel<false, 4, 1>, s);
  }
  if (rows) return launch_both(p, 64, few_fc1_kernel<8, 2>, 64, few_fc2_kernel<true, 4, 2>, s);
  return launch_both(p, 64, few_fc1_kernel<8, 2>, 128, few_fc2_kernel<false, 8, 2>, s);
}

extern "C" int mm_moe_few_int8(const int8_t* x, const float* x_scale, const int32_t* selected,
                               const float* routing_weights, const int8_t* w1, const float* w1_scale, const int8_t* w2,
                               const float* w2_scale, int64_t tokens, int32_t top_k, int32_t num_experts,
                               int32_t hidden, int32_t inter, int32_t act_kind, float situ_beta,
                               float situ_linear_beta, float clamp_limit, uint16_t* out, void* scratch,
                               size_t scratch_bytes, mm_stream_t stream) {
  MM_CHECK_ARG(few_sizes_ok(tokens, top_k, num_experts, hidden, inter), "mm_moe_few_int8: bad sizes");
  MM_CHECK_ARG(act_kind >= MM_ACT_SWIGLU && act_kind <= MM_ACT_CLAMP_SWIGLU, "mm_moe_few_int8: bad activation");
  if (tokens == 0) return MM_OK;
  const FewScratch f(tokens * top_k, hidden, inter, true);
  MM_CHECK_ARG(x && x_scale && selected && routing_weights && w1 && w1_scale && w2 && w2_scale && out && scratch,
               "mm_moe_few_int8: null pointer");
  if (scratch_bytes < f.bytes) {
    mm_set_error("mm_moe_few_int8: scratch needs %zu bytes", f.bytes);
    return MM_E_WS;
  }
  char* base = static_cast<char*>(scratch);
  FewArgs p{x, x_scale, selected, routing_weights, w1, w1_scale, w2, w2_scale, 0, 0,
            static_cast<int32_t>(tokens * top_k), top_k, num_experts, hidden, inter, static_cast<int32_t>(tokens),
            act_kind, situ_beta, situ_linear_beta, clamp_limit, base + f.act,
            reinterpret_cast<float*>(base + f.act_scale), reinterpret_cast<float*>(base + f.y),
            reinterpret_cast<int32_t*>(base + f.done), reinterpret_cast<bf16*>(out), 0, 0};
  const hipStream_t s = mm_hip_stream(stream);
  if (tokens <= 16) return launch_both(p, 32, few_fc1_int8_kernel<1>, 64, few_fc2_int8_kernel<1>, s);
  return launch_both(p, 32, few_fc1_int8_kernel<2>, 64, few_fc2_int8_kernel<2>, s);
}
