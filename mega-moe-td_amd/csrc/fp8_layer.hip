// The layer on E4M3 rows and E4M3 experts with a power-of-two scale for each
// block of 128 (fp8.h).
//
//   gu[i, :]  = x[token(i), :] W1[e]^T                 (held in fp32, e = expert of expert-major row i)
//   act[i, :] = act_fn(gate, up) * w[i], then E4M3 with a scale for each 128 columns
//   y[i, :]   = act[i, :] W2[e]^T                      (held in fp32)
//   out[t, :] = sum_j y[route_to_send[t k + j], :]     (fp32, slot order)
//
// gu and y are summed as fp8_tile.h says, gu of few activations in fp32 throughout.
// Routing tables and tile lists are those of the bf16 layer (a few rows need none). The experts' outputs
// stay in fp32 until the slots are summed: in bf16 each would be off by as much
// as the result is by its own rounding.
#include <algorithm>

#include "fp8_tile.h"

namespace {

struct LayerArgs {
  const uint8_t* x;     // rows [., K]
  const float* act;     // or, of a few rows' activation, in fp32
  const uint8_t* xs;    // their scales [., K / 128]
  const int32_t* rows;  // row of x of expert-major row i, or NULL: i
  const uint8_t* w;     // [E, C, K]
  const uint8_t* ws;    // [E, C / 128, K / 128]
  const float* weight;  // routing weight of row i (FC1)
  void* out;            // E4M3 [R, I] (FC1; a few rows: fp32) or fp32 [R, C]
  uint8_t* out_scale;   // [R, I / 128] (FC1)
  const TileList* tl;
  int32_t k, c, inter, act_kind;
  float beta, lbeta, limit;
};

// 32 bytes of a row's block, at any alignment: 16 and the 16 that lie 64 behind.
__device__ __forceinline__ i32x8 load32(const uint8_t* p) {
  i32x4 lo, hi;
  __builtin_memcpy(&lo, p, 16);
  __builtin_memcpy(&hi, p + 64, 16);
  return join32(lo, hi);
}

// ------------------------------------------------------------------ a few rows in all
// Where the ring's tiles below would leave most CUs idle: an expert's rows against
// 16 columns of the activation (the 16 gate and the 16 up channels) or 32 channels
// of the result. A workgroup belongs to a route and takes all rows of its expert if
// it is the expert's first: no tables, and a row is its route. The 4 waves share the
// blocks of K, 4 of them in flight in each, and join their sums in LDS; weights are
// the matrix instruction's rows, 16 of the expert's rows its columns. The activation
// passes in fp32: its 128 columns are in 8 workgroups, and each reader makes the same
// bytes of them in registers. FC1 sums in fp32 throughout: an activation that the
// E4M3 instruction's sums put on the other side of a rounding border, 1 in 10^3 to
// 10^4, is one of few here (one token: up to 0.005 of the result's norm).
// One token, H 2048, 8 experts of I 768: FC1 9.5 us for 25 MB, FC2 5.5 us for 13 MB,
// which the ring's tiles take 16 and 9 for, behind 6 us of routing.
constexpr int kFewRoutes = 256;

struct FewArgs {
  LayerArgs l;
  const int32_t* selected;
  int32_t routes, top_k, experts;
};

template <bool FC1>
__global__ __launch_bounds__(kFewRoutes) void fp8_few_kernel(FewArgs f) {
  using OP = std::conditional_t<FC1, Op16Wide, Op16>;
  constexpr int W = kFewRoutes / 64;
  __shared__ f32x4 sums[W - 1][2][64];
  __shared__ int32_t rows[kFewRoutes], counts[W];
  const LayerArgs& p = f.l;
  const int groups = FC1 ? p.inter / 16 : p.c / 32;
  const int route = blockIdx.x / groups, c0 = blockIdx.x % groups * (FC1 ? 16 : 32);
  const int expert = f.selected[route];
  if (expert < 0 || expert >= f.experts) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  const bool mine = static_cast<int>(threadIdx.x) < f.routes && f.selected[threadIdx.x] == expert;
  const uint64_t of_wave = __ballot(mine);
  if (lane == 0) counts[wave] = __popcll(of_wave);
  __syncthreads();
  int before = 0, count = 0;
#pragma unroll
  for (int v = 0; v < W; ++v) {
    before += v < wave ? counts[v] : 0;
    count += counts[v];
  }
  if (mine) rows[before + __popcll(of_wave & ((uint64_t(1) << lane) - 1))] = threadIdx.x;
  __syncthreads();
  if (rows[0] != route) return;
  const int kb = p.k / kBlock, c1 = FC1 ? p.inter + c0 : c0 + 16;
  const uint8_t* const w = p.w + static_cast<int64_t>(expert) * p.c * p.k;
  const uint8_t* const ws = p.ws + static_cast<int64_t>(expert) * (p.c / kBlock) * kb;
  const uint8_t* const w0 = w + static_cast<int64_t>(c0 + j) * p.k + 16 * q;
  const uint8_t* const w1 = w + static_cast<int64_t>(c1 + j) * p.k + 16 * q;
  const uint8_t* const s0 = ws + static_cast<int64_t>(c0 / kBlock) * kb;
  const uint8_t* const s1 = ws + static_cast<int64_t>(c1 / kBlock) * kb;
  for (int r = 0; r < count; r += 16) {
    const int i = rows[min(r + j, count - 1)];
    const int64_t row = FC1 ? i / f.top_k : i;
    const uint8_t* const x = p.x + row * p.k + 16 * q;
    const uint8_t* const xs = p.xs + row * kb;
    const float* const a = p.act + row * p.k + 16 * q;
    f32x4 acc[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
    auto steps = [&](auto blocks, int b) {
      constexpr int N = decltype(blocks)::value;
      i32x8 wv[N][2], xv[N];
      uint32_t sv[N][2], sx[N];
      f32x4 av[N][8];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int block = b + u * W;
        wv[u][0] = load32(w0 + block * kBlock);
        wv[u][1] = load32(w1 + block * kBlock);
        sv[u][0] = s0[block];
        sv[u][1] = s1[block];
        if constexpr (FC1) {
          xv[u] = load32(x + block * kBlock);
          sx[u] = xs[block];
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            av[u][i] = *reinterpret_cast<const f32x4*>(a + block * kBlock + i / 4 * 64 + i % 4 * 4);
        }
      }
#pragma unroll
      for (int u = 0; u < N; ++u) {
        if constexpr (!FC1) {
          uint32_t top = 0;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int v = 0; v < 4; ++v) top = max(top, abs_bits(av[u][i][v]));
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
          top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
          const BlockScale s(top);
          sx[u] = s.byte;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            xv[u][i] = static_cast<int>(s.pack4(av[u][i][0], av[u][i][1], av[u][i][2], av[u][i][3]));
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) acc[g] = OP::mac(OP::frag(wv[u][g]), OP::frag(xv[u]), acc[g], sv[u][g], sx[u]);
      }
    };
    int b = wave;
    for (; b + 3 * W < kb; b += 4 * W) steps(std::integral_constant<int, 4>{}, b);
    if (b + W < kb) {
      steps(std::integral_constant<int, 2>{}, b);
      b += 2 * W;
    }
    if (b < kb) steps(std::integral_constant<int, 1>{}, b);
    if (wave) {
      sums[wave - 1][0][lane] = acc[0];
      sums[wave - 1][1][lane] = acc[1];
    }
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int v = 0; v < W - 1; ++v) acc[g] += sums[v][g][lane];
      float* const out = static_cast<float*>(p.out) + static_cast<int64_t>(i) * (FC1 ? p.inter : p.c) + c0 + 4 * q;
      if (r + j >= count) {
      } else if constexpr (FC1) {
        const float weight = p.weight[i];
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = gated_act(p.act_kind, acc[0][k], acc[1][k], p.beta, p.lbeta, p.limit) * weight;
        *reinterpret_cast<f32x4*>(out) = v;
      } else {
        *reinterpret_cast<f32x4*>(out) = acc[0];
        *reinterpret_cast<f32x4*>(out + 16) = acc[1];
      }
    }
    __syncthreads();  // the sums are read
  }
}

// ------------------------------------------------------------------ many rows an expert
// Rows of K bytes, K a multiple of 128: 16-byte vectors of a stage, NT threads.
template <int ROWS, int NT>
struct RowPanel {
  static constexpr int PER = ROWS * 8 / NT;
  static_assert(PER * NT == ROWS * 8, "whole vectors");
  static constexpr bool CUTS = false;
  struct Stage {
    i32x4 d[PER];
  };
  const char* base;
  uint32_t off[PER];
  // row(r): index of the panel's r-th row
  template <class F>
  __device__ __forceinline__ RowPanel(const uint8_t* p, int K, const F& row) : base(reinterpret_cast<const char*>(p)) {
#pragma unroll
    for (int v = 0; v < PER; ++v) {
      const int c = v * NT + threadIdx.x;
      off[v] = static_cast<uint32_t>(row(c / 8)) * static_cast<uint32_t>(K) + c % 8 * 16;
    }
  }
  __device__ __forceinline__ void load_one(Stage& r, int v, int k) const {
    load_at(r.d[v], base + k, off[v]);
  }
  __device__ __forceinline__ void put_one(int8_t* lds, const Stage& r, int v) const {
    const int c = v * NT + threadIdx.x;
    *reinterpret_cast<i32x4*>(lds + slot_of(c / 8, c % 8)) = r.d[v];
  }
  __device__ __forceinline__ void load(Stage& r, int k) const {
#pragma unroll
    for (int v = 0; v < PER; ++v) load_one(r, v, k);
  }
  __device__ __forceinline__ void put(int8_t* lds, const Stage& r) const {
#pragma unroll
    for (int v = 0; v < PER; ++v) put_one(lds, r, v);
  }
  __device__ __forceinline__ void put_cut(int8_t*, int, int) const {}
};

constexpr int kWideRows = 64;

// One tile of 16 MI WM rows of an expert by 256 channels: with FC1 128 columns
// of the activation, a wave's channels gate and up of the same columns.
template <bool FC1, class OP, int MI, int WM, int WN, int PRE>
__device__ __forceinline__ void rows_tile(const LayerArgs& p, int8_t* lds, const int4& t, int cb) {
  constexpr int ROWS = kTile * MI, BM = ROWS * WM, BN = 256, NT = WM * WN * 64, COLS = BN / WN, NI = COLS / kTile;
  constexpr int GATE = NI / 2;  // tiles of gate channels (FC1)
  auto& smem = *reinterpret_cast<int8_t(*)[2][(BM + BN) * BK]>(lds);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
  const int kb = p.k / kBlock, r0 = t.y;
  const uint8_t* const ws = p.ws + static_cast<int64_t>(t.x) * (p.c / kBlock) * kb;
  // rows of x lie anywhere, those of act from the tile's first one on
  const int64_t base = FC1 ? 0 : r0;
  auto token = [&](int r) {
    const int i = min(r, t.z - 1 - r0);
    return FC1 ? p.rows[r0 + i] : i;
  };
  auto channel = [&](int r) {
    if (!FC1) return min(cb * BN + r, p.c - 1);
    const int w = r / COLS, c = r % COLS;
    return cb * kBlock + w * (COLS / 2) + c % (COLS / 2) + (c < COLS / 2 ? 0 : p.inter);
  };
  const RowPanel<BM, NT> pa(p.x + base * p.k, p.k, token);
  const RowPanel<BN, NT> pb(p.w + static_cast<int64_t>(t.x) * p.c * p.k, p.k, channel);
  const uint8_t* xs[MI];
#pragma unroll
  for (int i = 0; i < MI; ++i) xs[i] = p.xs + (base + token(wm * ROWS + i * kTile + token_of(lane))) * kb;
  auto sa = [&](int i, int block) -> uint32_t { return xs[i][block]; };
  const uint8_t* const sb0 = ws + static_cast<int64_t>(FC1 ? cb : min(cb * BN + wn * COLS, p.c - 1) / kBlock) * kb;
  const uint8_t* const sb1 = ws + static_cast<int64_t>(FC1 ? p.inter / kBlock + cb : 0) * kb;
  auto sb = [&](int h, int block) -> uint32_t { return h ? sb1[block] : sb0[block]; };
  f32x4 acc[MI][NI];
  tile_sums<OP, BM, BN, WM, WN, 1, PRE, FC1 ? 2 : 1>(smem, pa, pb, p.k, sa, sb, acc);
  __syncthreads();  // the stages are read

  if constexpr (FC1) {
    constexpr int PITCH = kBlock + 16;
    static_assert(BM * PITCH + WN * BM * 4 <= sizeof(smem), "epilogue staging");
    int8_t* const staged = lds;
    uint32_t* const tops = reinterpret_cast<uint32_t*>(lds + BM * PITCH);
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = wm * ROWS + i * kTile + token_of(lane);
      const float weight = p.weight[min(r0 + r, t.z - 1)];
      uint32_t top = 0;
#pragma unroll
      for (int j = 0; j < GATE; ++j)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float a = gated_act(p.act_kind, acc[i][j][v], acc[i][j + GATE][v], p.beta, p.lbeta, p.limit) * weight;
          acc[i][j][v] = a;
          top = max(top, abs_bits(a));
        }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      if (lane < 16) tops[wn * BM + r] = top;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MI; ++i) {
      const int r = wm * ROWS + i * kTile + token_of(lane);
      uint32_t top = 0;
#pragma unroll
      for (int w = 0; w < WN; ++w) top = max(top, tops[w * BM + r]);
      const BlockScale s(top);
      if (wn == 0 && lane < 16 && r0 + r < t.z)
        p.out_scale[static_cast<int64_t>(r0 + r) * (p.inter / kBlock) + cb] = static_cast<uint8_t>(s.byte);
#pragma unroll
      for (int j = 0; j < GATE; ++j)
        *reinterpret_cast<uint32_t*>(staged + r * PITCH + wn * (COLS / 2) + j * kTile + channel_of(lane)) =
            s.pack4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
    }
    __syncthreads();
    for (int v = threadIdx.x; v < BM * 8; v += NT) {
      const int r = v / 8, c = v % 8 * 16;
      if (r0 + r < t.z)
        *reinterpret_cast<i32x4*>(static_cast<uint8_t*>(p.out) + static_cast<int64_t>(r0 + r) * p.inter + cb * kBlock + c) =
            *reinterpret_cast<const i32x4*>(staged + r * PITCH + c);
    }
  } else {
    constexpr int PITCH = COLS * 4 + 16;
    static_assert(WM * WN * kTile * PITCH <= sizeof(smem), "epilogue staging");
    int8_t* const staged = lds + wave * (kTile * PITCH);
    struct {
      void* out;
      int64_t ldo;
      int32_t m, n;
    } to{p.out, p.c, t.z, p.c};
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<f32x4*>(staged + token_of(lane) * PITCH + (j * kTile + channel_of(lane)) * 4) = acc[i][j];
      store_rows<kTile, COLS, PITCH, float>(to, staged, r0 + wm * ROWS + i * kTile, cb * BN + wn * COLS);
    }
  }
}

// ------------------------------------------------------------------ weights streamed once
// Items of up to 160 rows of an expert (the 160-row tile list) by 256 channels, one
// after another in each of the chip's CUs. A stage is a block of K: the weights'
// and the rows' bytes are copied straight to LDS, with their scale bytes, into a
// ring of three; 2 x 4 waves multiply. A buffer is copied into again as soon as its
// last fragment is read, and the copies run on into the next item: with a
// workgroup for each item, alone on its CU by its LDS, the memory idled for 8 us in
// front of an item, 7 behind it and 8 between workgroups, of 110 (4096 tokens, H
// 7168, E 256 top-8). There FC1 has 7.5 GB of weights and takes 1.62 ms, 4.6 TB/s,
// with LDS busy for 20% of it and the matrix unit for 31%; 64 experts of 4 rows take
// 277 us for 1.9 GB, 6.8 TB/s (with WIDE 290).
//
// The compiler does not know of the copies: wait_copies and a barrier stand in front
// of what reads them. A load that it knows waits for all of them: row numbers and
// tiles come through the scalar cache, routing weights by a copy. What is left are
// registers that it spills and loads again: in FC2 in front of every item and in the
// last stage of those of more than 128 rows, in FC1 (not WIDE) behind the last stage
// of those; there the ring is empty for a moment.
typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ uint32_t lds_offset(const int8_t* p) {
  return __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void*)(p))));
}
// A wave's copy of 16 bytes a lane, lane l's to `lds` + 16 l. (m0 cannot be declared as written: it is the compiler's
// own, which keeps nothing in it and sets it in front of each of its uses, of which these kernels have none.)
__device__ __forceinline__ void copy_lines(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory");
}
// The same of bytes that no other workgroup reads soon: they are the first that the caches let go.
__device__ __forceinline__ void copy_lines_once(const char* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(base), "s"(lds) : "memory");
}
// Of a byte each in the first 26 lanes, lane l's to the word at `lds` + 4 l.
__device__ __forceinline__ void copy_scales(const uint8_t* p, uint32_t lds) {
  uint64_t lanes;
  asm volatile("s_and_saveexec_b64 %0, %3\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, off\n\ts_mov_b64 exec, %0"
               : "=&s"(lanes) : "v"(p), "s"(lds), "s"(uint64_t(0x3ffffff)) : "memory", "scc");
}
// Of a float a lane.
__device__ __forceinline__ void copy_float(const float* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(p), "s"(lds) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_copies() {  // until N of the wave's are left
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | (0x7 << 4) | (0xF << 8));
}

typedef int i32x8s __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x4 scalar_load4(const void* p) {
  i32x4 v;
  asm volatile("s_load_dwordx4 %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=s"(v) : "s"(p) : "memory");
  return v;
}
__device__ __forceinline__ i32x8s scalar_load8(const void* p) {
  i32x8s v;
  asm volatile("s_load_dwordx8 %0, %1, 0x0\n\ts_waitcnt lgkmcnt(0)" : "=s"(v) : "s"(p) : "memory");
  return v;
}
__device__ __forceinline__ int pick(const i32x8s& v, int i) {
  int r = v[0];
#pragma unroll
  for (int k = 1; k < 8; ++k) r = i == k ? v[k] : r;
  return r;
}

namespace ring {
constexpr int kRows = kStreamRows, kChannels = 256, kDepth = 3;
constexpr int kPanels = (kRows + kChannels) * BK;  // bytes of a stage's rows and weights, in copies of 8 rows (1 KB)
constexpr int kWaveScales = 32;                    // words of a wave's scales: its 24 rows', then the channels' two
constexpr int kStage = kPanels + 8 * kWaveScales * 4;
constexpr int kWeights = kDepth * kStage;  // routing weights of 192 rows
constexpr int kBytes = kWeights + 192 * 4;
constexpr int kCopies = 4 + 3 + 1;  // a wave and stage: of weights, of rows, of scales
static_assert(kBytes <= 160 * 1024, "fits LDS");
// where the scale of row r is: the wave that copies the row copies it too
__device__ __forceinline__ int scale_slot(int r) { return (r >> 3 & 7) * kWaveScales + (r >> 6) * 8 + (r & 7); }
}  // namespace ring

// ONCE: weights that the caches need not keep. WIDE (FC1): sums in fp32 throughout.
template <bool FC1, bool ONCE, bool WIDE>
struct Ring {
  struct Item {
    const char* w;      // its first channel's weights
    const char* x;      // the rows' base
    int r0, rows, c0;   // expert-major rows from r0 on; first channel (FC1: column of the activation)
    uint32_t off[3];    // the lane's bytes of the wave's copies of rows
    const uint8_t* scale;  // the lane's scale, of block 0
  };
  const LayerArgs& p;
  int8_t* const lds;
  const uint32_t lds0;
  const int lane, wave, wm, wn, kb, stages, cblocks, step, count;
  uint32_t w_off[4];
  Item cur, next;
  int buf;

  __device__ __forceinline__ Ring(const LayerArgs& args, int8_t* l)
      : p(args), lds(l), lds0(lds_offset(l)), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
        wm(wave / 4), wn(wave % 4), kb(args.k / kBlock),
        stages(max(kb, ring::kDepth)),  // so that no item is passed over; a stage past K is not multiplied
        cblocks(FC1 ? args.inter / kBlock : (args.c + 255) / 256), step(gridDim.x / 8),
        count(__builtin_amdgcn_readfirstlane(args.tl->count)), buf(0) {
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const int r = (v * 8 + wave) * 8 + lane / 8, in = r % 64;
      // a wave's 64 channels: 32 of gate and the 32 of up for the same columns (FC1)
      const int c = FC1 ? r / 64 * 32 + in % 32 + (in < 32 ? 0 : p.inter) : min(r, p.c - 1);
      w_off[v] = static_cast<uint32_t>(c) * static_cast<uint32_t>(p.k) + slot(r);
    }
  }
  // what slot_of keeps where this lane's 16 bytes of row r go
  __device__ __forceinline__ uint32_t slot(int r) const { return ((lane & 7) ^ (r >> 1 & 7)) << 4; }
  // XCD x takes the tiles x, x + 8, ... with all their channels, so that an expert's
  // rows come from one L2; its workgroups take them in turn
  __device__ __forceinline__ int tile_of(int n) const { return n / cblocks * 8 + static_cast<int>(blockIdx.x & 7); }

  __device__ __forceinline__ void take(Item& it, int n) const {
    const i32x4 t = scalar_load4(p.tl->tiles + tile_of(n));
    const int cb = n % cblocks;
    it.r0 = t[1];
    it.rows = t[2] - t[1];
    // the last 256 channels again where they are not a whole run
    it.c0 = FC1 ? cb * kBlock : min(cb * 256, max(p.c - 256, 0));
    it.w = reinterpret_cast<const char*>(p.w) + (static_cast<int64_t>(t[0]) * p.c + it.c0) * p.k;
    it.x = reinterpret_cast<const char*>(p.x) + (FC1 ? 0 : static_cast<int64_t>(it.r0) * p.k);
    int scale_row = 0;
#pragma unroll
    for (int v = 0; v < 3; ++v) {
      const int r = min(v * 8 + wave, ring::kRows / 8 - 1) * 8;  // first row of the copy
      // eight row numbers that hold it (those past the last row are the scratch's next bytes, and not picked)
      const int first = min(r, (it.rows - 1) & ~7);
      const i32x8s ids = FC1 ? scalar_load8(p.rows + it.r0 + first) : i32x8s{0, 1, 2, 3, 4, 5, 6, 7} + first;
      it.off[v] = static_cast<uint32_t>(pick(ids, min(r + lane / 8, it.rows - 1) - first)) * static_cast<uint32_t>(p.k) +
                  slot(r + lane / 8);
      const int row = pick(ids, min(r + lane % 8, it.rows - 1) - first);
      if (lane / 8 == v) scale_row = row;
    }
    const int h = lane - 24;  // 0 and 1: of gate and up, or of the run's two blocks of channels
    const uint8_t* const ws = p.ws + static_cast<int64_t>(t[0]) * (p.c / kBlock) * kb;
    const int channels = FC1 ? cb + (h & 1) * (p.inter / kBlock) : min(it.c0 / kBlock + (h & 1), p.c / kBlock - 1);
    it.scale = h < 0 ? p.xs + ((FC1 ? 0 : static_cast<int64_t>(it.r0)) + scale_row) * kb : ws + static_cast<int64_t>(channels) * kb;
  }

  // Copies stage s of the current item, or of the next one behind its last.
  __device__ __forceinline__ void copy(int s, int to_buf) const {
    const bool in = s < stages;
    const int block = min(in ? s : s - stages, kb - 1);
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds0 + to_buf * ring::kStage);
    const char* const w = (in ? cur.w : next.w) + block * BK;
    const char* const x = (in ? cur.x : next.x) + block * BK;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const uint32_t panel = to + ring::kRows * BK + (v * 8 + wave) * 1024;
      if constexpr (ONCE)
        copy_lines_once(w, w_off[v], panel);
      else
        copy_lines(w, w_off[v], panel);
    }
#pragma unroll
    for (int v = 0; v < 3; ++v)
      copy_lines(x, in ? cur.off[v] : next.off[v], to + min(v * 8 + wave, ring::kRows / 8 - 1) * 1024);
    copy_scales((in ? cur.scale : next.scale) + block, to + ring::kPanels + wave * (ring::kWaveScales * 4));
  }
  __device__ __forceinline__ void copy_weights() const {  // of the current item's rows
    const int w = wave % 3;
    if constexpr (FC1) copy_float(p.weight + cur.r0 + min(w * 64 + lane, cur.rows - 1), lds0 + ring::kWeights + w * 256);
  }

  // The current item's sums for up to 32 MI rows, and what becomes of them. Leaves
  // the last stage's buffer to be copied into.
  template <int MI>
  __device__ __forceinline__ void run() {
    constexpr int NI = 4, ROWS = kTile * MI;
    int id = lane;  // kept from the other heights' addresses, which would all be held in registers
    asm volatile("" : "+v"(id));
    const int j = id & 15, q = id >> 4;
    auto bytes = [&](const int8_t* panel, int row) __attribute__((always_inline)) {
      return join32(*reinterpret_cast<const i32x4*>(panel + slot_of(row, q)),
                    *reinterpret_cast<const i32x4*>(panel + slot_of(row, 4 + q)));
    };
    auto bytes_a = [&](const int8_t* b, int i) __attribute__((always_inline)) { return bytes(b, wm * ROWS + i * kTile + j); };
    auto bytes_b = [&](const int8_t* b, int c) __attribute__((always_inline)) {
      return bytes(b + ring::kRows * BK, (wn * NI + c) * kTile + j);
    };
    int at[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) at[i] = ring::scale_slot(wm * ROWS + i * kTile + j);
    i32x8 fa[MI], fb;
    uint32_t as[MI], bs[2], as_next[MI], bs_next[2];
    auto scales = [&](const int8_t* b, uint32_t (&a)[MI], uint32_t (&c)[2]) __attribute__((always_inline)) {
      const uint32_t* const from = reinterpret_cast<const uint32_t*>(b + ring::kPanels);
#pragma unroll
      for (int i = 0; i < MI; ++i) a[i] = from[at[i]];
#pragma unroll
      for (int h = 0; h < 2; ++h) c[h] = from[wave * ring::kWaveScales + 24 + h];
    };
    f32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int c = 0; c < NI; ++c) acc[i][c] = f32x4{0, 0, 0, 0};
    if constexpr (WIDE && MI > 2) {
      // The next stage's bytes and this one's in bf16 do not fit the registers together with so many sums: here a
      // stage is read when it is there, its channels kept in bf16, its rows 16 by 16.
      for (int s = 0; s < stages; ++s) {
        const int8_t* const now = lds + buf * ring::kStage;
        if (s < kb) {
          scales(now, as, bs);
          Op16Wide::Frag fw[NI];
#pragma unroll
          for (int c = 0; c < NI; ++c) fw[c] = Op16Wide::frag(bytes_b(now, c));
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            const Op16Wide::Frag wide = Op16Wide::frag(bytes_a(now, i));
#pragma unroll
            for (int c = 0; c < NI; ++c) acc[i][c] = Op16Wide::mac(fw[c], wide, acc[i][c], bs[c / 2], as[i]);
          }
        }
        wait_copies<(ring::kDepth - 2) * ring::kCopies>();
        __syncthreads();
        if (s + 1 < stages) {
          copy(s + ring::kDepth, buf);
          buf = buf + 1 == ring::kDepth ? 0 : buf + 1;
        }
      }
      finish<MI>(acc, lds + buf * ring::kStage);
      return;
    }
    const int8_t* b = lds + buf * ring::kStage;
#pragma unroll
    for (int i = 0; i < MI; ++i) fa[i] = bytes_a(b, i);
    fb = bytes_b(b, 0);
    scales(b, as, bs);
    auto stage = [&](int s, auto last) __attribute__((always_inline)) {
      constexpr bool LAST = decltype(last)::value;
      const int next_buf = buf + 1 == ring::kDepth ? 0 : buf + 1;
      const int8_t* const now = lds + buf * ring::kStage;
      const int8_t* const nxt = lds + next_buf * ring::kStage;
      Op16Wide::Frag wide[WIDE ? MI : 1];
      if constexpr (WIDE) {
#pragma unroll
        for (int i = 0; i < MI; ++i) wide[i] = Op16Wide::frag(fa[i]);
      }
#pragma unroll
      for (int c = 0; c < NI; ++c) {
        const bool tail = c == NI - 1;
        if (tail) {  // every wave has read this stage, and its copies of the next have arrived
          wait_copies<(ring::kDepth - 2) * ring::kCopies>();
          __syncthreads();
          if constexpr (!LAST) {
            copy(s + ring::kDepth, buf);
            scales(nxt, as_next, bs_next);
          }
        }
        i32x8 fb_next = fb;
        if (!(tail && LAST)) fb_next = tail ? bytes_b(nxt, 0) : bytes_b(now, c + 1);
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          if constexpr (!WIDE) {
            acc[i][c] = Op16::mac(fb, fa[i], acc[i][c], bs[FC1 ? c / 2 : wn / 2], as[i]);
            if (tail && !LAST) fa[i] = bytes_a(nxt, i);
          }
        }
        if constexpr (WIDE) {
          const Op16Wide::Frag fw = Op16Wide::frag(fb);
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            acc[i][c] = Op16Wide::mac(fw, wide[i], acc[i][c], bs[c / 2], as[i]);
            if (tail && !LAST) fa[i] = bytes_a(nxt, i);
          }
        } else {
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS read
#pragma unroll
          for (int i = 0; i < MI; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
            if (tail) __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        fb = fb_next;
      }
      if constexpr (!LAST) {
#pragma unroll
        for (int i = 0; i < MI; ++i) as[i] = as_next[i];
        bs[0] = bs_next[0];
        bs[1] = bs_next[1];
        buf = next_buf;
      }
    };
    for (int s = 0; s + 1 < kb; ++s) stage(s, std::false_type{});
    if (kb == stages) {
      stage(kb - 1, std::true_type{});
    } else {  // stages past K: their copies are waited for, and the next ones begun
      stage(kb - 1, std::false_type{});
      for (int s = kb; s < stages; ++s) {
        wait_copies<(ring::kDepth - 2) * ring::kCopies>();
        __syncthreads();
        if (s + 1 < stages) {
          copy(s + ring::kDepth, buf);
          buf = buf + 1 == ring::kDepth ? 0 : buf + 1;
        }
      }
    }
    finish<MI>(acc, lds + buf * ring::kStage);
  }

  // `free`: a stage's bytes of LDS that nothing is copied into
  template <int MI>
  __device__ __forceinline__ void finish(f32x4 (&acc)[MI][4], int8_t* free) {
    constexpr int ROWS = kTile * MI, BM = 2 * ROWS, NI = 4;
    int lane = this->lane;
    asm volatile("" : "+v"(lane));
    if constexpr (FC1) {
      constexpr int PITCH = kBlock + 16;
      static_assert(BM * PITCH + 4 * BM * 4 <= ring::kStage, "epilogue staging");
      const float* const weights = reinterpret_cast<const float*>(lds + ring::kWeights);
      uint32_t* const tops = reinterpret_cast<uint32_t*>(free + BM * PITCH);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = wm * ROWS + i * kTile + token_of(lane);
        const float weight = weights[r];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            const float a = gated_act(p.act_kind, acc[i][c][v], acc[i][c + 2][v], p.beta, p.lbeta, p.limit) * weight;
            acc[i][c][v] = a;
            top = max(top, abs_bits(a));
          }
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
        if (lane < 16) tops[wn * BM + r] = top;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int r = wm * ROWS + i * kTile + token_of(lane);
        uint32_t top = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = max(top, tops[w * BM + r]);
        const BlockScale s(top);
        if (wn == 0 && lane < 16 && r < cur.rows)
          p.out_scale[static_cast<int64_t>(cur.r0 + r) * (p.inter / kBlock) + cur.c0 / kBlock] = static_cast<uint8_t>(s.byte);
#pragma unroll
        for (int c = 0; c < 2; ++c)
          *reinterpret_cast<uint32_t*>(free + r * PITCH + wn * 32 + c * kTile + channel_of(lane)) =
              s.pack4(acc[i][c][0], acc[i][c][1], acc[i][c][2], acc[i][c][3]);
      }
      __syncthreads();
      for (int v = wave * 64 + lane; v < BM * 8; v += 512) {
        const int r = v / 8, c = v % 8 * 16;
        if (r < cur.rows)
          *reinterpret_cast<i32x4*>(static_cast<uint8_t*>(p.out) + static_cast<int64_t>(cur.r0 + r) * p.inter + cur.c0 + c) =
              *reinterpret_cast<const i32x4*>(free + r * PITCH + c);
      }
    } else {
      constexpr int COLS = NI * kTile, PITCH = COLS * 4 + 16;
      static_assert(8 * kTile * PITCH <= ring::kStage, "epilogue staging");
      int8_t* const staged = free + wave * (kTile * PITCH);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int c = 0; c < NI; ++c)
          *reinterpret_cast<f32x4*>(staged + token_of(lane) * PITCH + (c * kTile + channel_of(lane)) * 4) = acc[i][c];
        const int first = wm * ROWS + i * kTile, col = cur.c0 + wn * COLS + (lane & 15) * 4;
#pragma unroll
        for (int v = 0; v < 4; ++v) {  // 4 rows a wave at a time
          const int r = v * 4 + (lane >> 4);
          const f32x4 sum = *reinterpret_cast<const f32x4*>(staged + r * PITCH + (lane & 15) * 16);
          if (first + r < cur.rows && col < p.c) {
            f32x4* const to = reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + static_cast<int64_t>(cur.r0 + first + r) * p.c + col);
            if constexpr (ONCE)  // past the caches too (0.94 GB: 0.88 ms, 0.92 through them, and the slots' sum 0.20 and 0.23)
              __builtin_nontemporal_store(sum, to);
            else
              *to = sum;
          }
        }
      }
    }
  }

  __device__ __forceinline__ void all() {
    int n = blockIdx.x >> 3;
    if (tile_of(n) >= count) return;
    take(cur, n);
    for (int s = 0; s < ring::kDepth; ++s) copy(s, s);
    copy_weights();
    wait_copies<(ring::kDepth - 1) * ring::kCopies>();
    __syncthreads();
    for (;;) {
      const bool more = tile_of(n + step) < count;
      take(next, more ? n + step : n);
      if (cur.rows <= 32)
        run<1>();
      else if (cur.rows <= 64)
        run<2>();
      else if (cur.rows <= 128)
        run<4>();
      else
        run<5>();
      if (!more) break;
      __syncthreads();  // the buffer that the epilogue used
      copy(stages - 1 + ring::kDepth, buf);
      buf = buf + 1 == ring::kDepth ? 0 : buf + 1;
      cur = next;
      copy_weights();
      n += step;
    }
    wait_copies<0>();  // nothing is copied into LDS that another workgroup has by then
  }
};

template <bool FC1, bool ONCE, bool WIDE>
__global__ __launch_bounds__(512) void fp8_ring_kernel(LayerArgs p) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[ring::kBytes];
  Ring<FC1, ONCE, WIDE>(p, lds).all();
}

// Experts of many rows, whose weights several tiles of the 256-row list read: tile
// m runs on XCD m % 8 with all its channels, so that its rows come from one L2.
// WIDE (FC1): sums in fp32 throughout, a workgroup for each 64 of a tile's rows.
template <bool FC1, bool WIDE>
__global__ __launch_bounds__(512) void fp8_rows_kernel(LayerArgs p) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[2 * ((WIDE ? kWideRows : 256) + 256) * BK];
  constexpr int parts = WIDE ? 256 / kWideRows : 1;
  const int cblocks = FC1 ? p.inter / kBlock : (p.c + 255) / 256;
  const int slot = blockIdx.x >> 3, tile = slot / (cblocks * parts) * 8 + (blockIdx.x & 7);
  const int cb = slot % (cblocks * parts) / parts, part = slot % parts;
  if (tile >= p.tl->count) return;
  int4 t = p.tl->tiles[tile];
  if constexpr (WIDE) {
    t.y += part * kWideRows;
    t.z = min(t.z, t.y + kWideRows);
    if (t.y < t.z) rows_tile<FC1, Op16Wide, 2, 2, 4, 2>(p, lds, t, cb);
  } else if (t.z - t.y <= 128) {
    rows_tile<FC1, Op16, 2, 4, 2, 1>(p, lds, t, cb);
  } else {
    rows_tile<FC1, Op16, 4, 4, 2, 1>(p, lds, t, cb);
  }
}

// out[t, :] = sum of the token's slots in slot order; a thread has 8 columns and
// loads 4 slots at once (one token: 2.9 us, and 5.6 with one behind another).
// Slots name their rows of y (-1: none) or, with ROUTES, their experts: then a
// slot's row is its route. 4096 tokens of 8 slots, H 7168: 0.2 ms for 1 GB, 5 TB/s.
template <bool ROUTES>
__global__ __launch_bounds__(256) void fp8_combine_kernel(const float* y, const int32_t* slot, int32_t experts, uint32_t tokens,
                                                          int32_t top_k, int32_t hidden, uint16_t* out) {
  const uint32_t chunks = hidden / 8, total = tokens * chunks;  // below 2^29
  for (uint32_t v = blockIdx.x * 256 + threadIdx.x; v < total; v += gridDim.x * 256) {
    const uint32_t token = v / chunks, c = (v - token * chunks) * 8;
    const int64_t first = static_cast<int64_t>(token) * top_k;
    float sum[8] = {};
    auto slots = [&](auto count, int j) __attribute__((always_inline)) {
      constexpr int N = decltype(count)::value;
      int32_t row[N];
      f32x4 a[N], b[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        row[n] = slot[first + j + n];
        if constexpr (ROUTES) row[n] = row[n] >= 0 && row[n] < experts ? static_cast<int32_t>(first) + j + n : -1;
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {  // a slot of no expert: a row that is not added
        const f32x4* from = reinterpret_cast<const f32x4*>(y + static_cast<int64_t>(max(row[n], 0)) * hidden + c);
        a[n] = from[0];
        b[n] = from[1];
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum[i] = row[n] < 0 ? sum[i] : sum[i] + a[n][i];
          sum[4 + i] = row[n] < 0 ? sum[4 + i] : sum[4 + i] + b[n][i];
        }
      }
    };
    int j = 0;
    for (; j + 4 <= top_k; j += 4) slots(std::integral_constant<int, 4>{}, j);
    for (; j < top_k; ++j) slots(std::integral_constant<int, 1>{}, j);
    *reinterpret_cast<uint4*>(out + static_cast<int64_t>(token) * hidden + c) =
        make_uint4(pack_bf16x2(sum[0], sum[1]), pack_bf16x2(sum[2], sum[3]), pack_bf16x2(sum[4], sum[5]), pack_bf16x2(sum[6], sum[7]));
  }
}

// ------------------------------------------------------------------ the whole layer
struct Carver {
  char* base;
  size_t used = 0;
  template <class T>
  T* take(size_t bytes) {
    T* p = reinterpret_cast<T*>(base + used);
    used += mm_align_up(bytes, 256);
    return p;
  }
};

// Bytes of the weights that R rows read at most.
int64_t weight_bytes(int64_t R, int E, int hidden, int inter) { return std::min<int64_t>(R, E) * 3 * inter * hidden; }

// Up to 256 routes, on average up to 16 an expert, are better off in fp8_few_kernel, whose workgroups are many and
// short, where they are no more than 64 or read no more than 512 MB of weights: H 2048, I 768, E 128 top-8 one token
// 17.5 us (33 with the ring), 4 tokens 44 (47), 8 tokens 71 (72), 32 tokens (604 MB) 160 (118); H 7168, I 2048, E 64
// one token 80 (88), 2 tokens 136 (137), 4 tokens 229 (233), 16 tokens (2.8 GB) 500 (431).
bool few_rows(int64_t R, int E, int hidden, int inter) {
  return R <= kFewRoutes && R <= int64_t(16) * E && (R <= 64 || weight_bytes(R, E, hidden, inter) <= int64_t(512) << 20);
}

struct Scratch {
  int32_t *counts, *offsets, *send_route, *send_token, *route_to_send;
  float* weight_perm;
  void *tiles, *route_ws;
  uint8_t *act, *act_scale;  // act of a few rows: fp32
  float* y;
  size_t tiles_bytes, route_ws_bytes, bytes;

  Scratch(void* base, int64_t R, int E, int hidden, int inter) {
    Carver c{static_cast<char*>(base)};
    const size_t r = static_cast<size_t>(R);
    const bool few = few_rows(R, E, hidden, inter);  // which needs no tables
    tiles_bytes = mm_tile_lists_bytes(R, E);
    route_ws_bytes = mm_route_workspace_bytes(R, E);
    y = c.take<float>(r * hidden * 4);
    act = c.take<uint8_t>(r * inter * (few ? 4 : 1));
    if (!few) {
      act_scale = c.take<uint8_t>(r * (inter / kBlock));
      route_ws = c.take<void>(route_ws_bytes);
      tiles = c.take<void>(tiles_bytes);
      counts = c.take<int32_t>(static_cast<size_t>(E) * 4);
      offsets = c.take<int32_t>(static_cast<size_t>(E + 1) * 4);
      send_route = c.take<int32_t>(r * 4);
      send_token = c.take<int32_t>(r * 4);
      route_to_send = c.take<int32_t>(r * 4);
      weight_perm = c.take<float>(r * 4);
    }
    bytes = c.used;
  }
};

constexpr int kMaxDim = 1 << 20;

// The rows of x, and an expert's weights, have 32-bit offsets.
bool layer_sizes_ok(int64_t tokens, int32_t top_k, int32_t E, int32_t hidden, int32_t inter) {
  constexpr int64_t most = int64_t(1) << 32;
  return tokens >= 0 && top_k > 0 && top_k <= 64 && E > 0 && E <= 32768 && hidden > 0 && inter > 0 &&
         hidden <= kMaxDim && inter <= kMaxDim && hidden % kBlock == 0 && inter % kBlock == 0 &&
         tokens < (int64_t(1) << 31) / top_k && tokens * hidden < most &&
         int64_t(2) * inter * hidden < most;
}

template <class Args>
int launch(void (*kernel)(Args), int64_t blocks, int threads, const Args& p, hipStream_t s) {
  MM_CHECK_ARG(blocks * threads < (int64_t(1) << 32), "mm_moe_fp8: too many tiles");
  kernel<<<static_cast<uint32_t>(blocks), threads, 0, s>>>(p);
  return mm_check_launch("mm_moe_fp8");
}

}  // namespace

extern "C" size_t mm_moe_fp8_scratch_bytes(int64_t tokens, int32_t top_k, int32_t num_experts, int32_t hidden,
                                           int32_t inter) {
  if (!layer_sizes_ok(tokens, top_k, num_experts, hidden, inter)) return 0;
  return Scratch(nullptr, tokens * top_k, num_experts, hidden, inter).bytes;
}

extern "C" int mm_moe_fp8(const uint8_t* x, const uint8_t* x_scale, const int32_t* selected,
                          const float* routing_weights, const uint8_t* w1, const uint8_t* w1_scale, const uint8_t* w2,
                          const uint8_t* w2_scale, int64_t tokens, int32_t top_k, int32_t num_experts, int32_t hidden,
                          int32_t inter, int32_t act_kind, float situ_beta, float situ_linear_beta, float clamp_limit,
                          uint16_t* out, void* scratch, size_t scratch_bytes, mm_stream_t stream) {
  MM_CHECK_ARG(layer_sizes_ok(tokens, top_k, num_experts, hidden, inter), "mm_moe_fp8: bad sizes");
  MM_CHECK_ARG(act_kind >= 0 && act_kind <= 2, "mm_moe_fp8: bad act_kind");
  if (tokens == 0) return MM_OK;
  const int E = num_experts;
  const int64_t R = tokens * top_k;
  const Scratch s(scratch, R, E, hidden, inter);
  MM_CHECK_ARG(x && x_scale && selected && routing_weights && w1 && w1_scale && w2 && w2_scale && out,
               "mm_moe_fp8: null pointer");
  MM_CHECK_ARG(((reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(x) |
                 reinterpret_cast<uintptr_t>(w1) | reinterpret_cast<uintptr_t>(w2)) & 15) == 0,
               "mm_moe_fp8: x, w1, w2, out and scratch must be 16-byte aligned");
  if (!scratch || scratch_bytes < s.bytes) {
    mm_set_error("mm_moe_fp8: scratch needs %zu bytes", s.bytes);
    return MM_E_WS;
  }
  const hipStream_t hs = mm_hip_stream(stream);
  const int64_t groups = std::min<int64_t>((tokens * (hidden / 8) + 255) / 256, 65536);  // of the slots' sums
  if (few_rows(R, E, hidden, inter)) {
    float* const act = reinterpret_cast<float*>(s.act);
    const FewArgs fc1{{x, nullptr, x_scale, nullptr, w1, w1_scale, routing_weights, act, nullptr, nullptr, hidden, 2 * inter, inter,
                       act_kind, situ_beta, situ_linear_beta, clamp_limit},
                      selected, static_cast<int32_t>(R), top_k, E};
    const FewArgs fc2{{nullptr, act, nullptr, nullptr, w2, w2_scale, nullptr, s.y, nullptr, nullptr, inter, hidden, inter, 0, 0, 0, 0},
                      selected, static_cast<int32_t>(R), top_k, E};
    int rc = launch(fp8_few_kernel<true>, R * (inter / 16), kFewRoutes, fc1, hs);
    if (!rc) rc = launch(fp8_few_kernel<false>, R * (hidden / 32), kFewRoutes, fc2, hs);
    if (rc) return rc;
    fp8_combine_kernel<true><<<static_cast<uint32_t>(groups), 256, 0, hs>>>(s.y, selected, E, static_cast<uint32_t>(tokens), top_k,
                                                                            hidden, out);
    return mm_check_launch("fp8_combine_kernel");
  }
  int rc = mm_route_tiles(selected, R, top_k, E, routing_weights, s.counts, s.offsets, s.send_route, s.send_token,
                          s.route_to_send, s.weight_perm, s.tiles, s.tiles_bytes, s.route_ws, s.route_ws_bytes, stream);
  if (rc) return rc;
  const int64_t mean = (R + E - 1) / E;  // rows an expert
  const LayerArgs fc1{x, nullptr, x_scale, s.send_token, w1, w1_scale, s.weight_perm, s.act, s.act_scale, nullptr, hidden, 2 * inter,
                      inter, act_kind, situ_beta, situ_linear_beta, clamp_limit};
  const LayerArgs fc2{s.act, nullptr, s.act_scale, nullptr, w2, w2_scale, nullptr, s.y, nullptr, nullptr, inter, hidden, inter, 0, 0, 0, 0};
  // Weights that the last-level cache (256 MB) cannot hold from one call to the
  // next pass it by: 604 MB of them in 75 us instead of 84 (FC1), 2.8 GB in 277
  // instead of 306, but 38 MB in 19 instead of 16.
  const bool once = weight_bytes(R, E, hidden, inter) > int64_t(192) << 20;
  auto run = [&](void (*ring)(LayerArgs), void (*rows)(LayerArgs), LayerArgs p, int64_t cblocks) {
    const int height = ring ? kStreamRows : 256;
    const int64_t items = (mm_max_m_tiles(R, E, height) + 7) / 8 * 8 * cblocks;
    p.tl = mm_tile_list_of(s.tiles, R, E, height);
    // the ring takes a CU's items in turn
    return launch(ring ? ring : rows, ring ? std::min<int64_t>(items, 256) : items, 512, p, hs);
  };
  // By rows an expert on average: above 128 many have more than the ring's 160 and would stream their weights twice
  // (H 7168, I 2048, E 16: 120 rows 179 us with the ring and 196 in tiles of 256, 150 rows 282 and 219, 200 rows 343
  // and 230, 2000 rows 2.23 and 1.67 ms)
  const bool streamed = mean <= 128;
  // The E4M3 instruction's sums are 1.4e-5 off, which moves 1 of 3000 activations by a step of E4M3, and the scale of 1
  // of 25000 blocks: among many 0.0017 of the result's norm, as much as bf16 rounds. Among few it can be several times
  // that (800 rows, I 128: 0.007 once in ten), so few are summed in fp32 throughout: up to 2 million where FC1 waits for
  // weights anyhow (64 experts of 4 rows, H 7168: 468 us, 450 otherwise; an item of more than 64 rows takes as long to
  // multiply as to load: 8 experts of 62 rows, H 7168, 182 and 127), else up to half a million (16 experts of 80
  // rows, H 1024, I 256: 36 and 37 us, but 8 of 80, H 4096, I 1536: 125 and 78).
  const bool wide = R * inter <= int64_t(1) << (mean <= 64 ? 21 : 19);
  const int64_t fc1_cblocks = inter / kBlock, fc2_cblocks = (hidden + 255) / 256;
  if (wide && mean <= 64)
    rc = run(once ? fp8_ring_kernel<true, true, true> : fp8_ring_kernel<true, false, true>, nullptr, fc1, fc1_cblocks);
  else if (wide)
    rc = run(nullptr, fp8_rows_kernel<true, true>, fc1, fc1_cblocks * (256 / kWideRows));
  else if (streamed)
    rc = run(once ? fp8_ring_kernel<true, true, false> : fp8_ring_kernel<true, false, false>, nullptr, fc1, fc1_cblocks);
  else
    rc = run(nullptr, fp8_rows_kernel<true, false>, fc1, fc1_cblocks);
  if (rc) return rc;
  if (streamed)
    rc = run(once ? fp8_ring_kernel<false, true, false> : fp8_ring_kernel<false, false, false>, nullptr, fc2, fc2_cblocks);
  else
    rc = run(nullptr, fp8_rows_kernel<false, false>, fc2, fc2_cblocks);
  if (rc) return rc;
  fp8_combine_kernel<false><<<static_cast<uint32_t>(groups), 256, 0, hs>>>(s.y, s.route_to_send, E, static_cast<uint32_t>(tokens),
                                                                           top_k, hidden, out);
  return mm_check_launch("fp8_combine_kernel");
}
