// The layer on E4M3 rows and E4M3 experts with a power-of-two scale for each
// block of 128 (fp8.h).
//
//   gu[i, :]  = x[token(i), :] W1[e]^T                 (fp32, e = expert of expert-major row i)
//   act[i, :] = act_fn(gate, up) * w[i], then E4M3 with a scale for each 128 columns
//   y[i, :]   = act[i, :] W2[e]^T                      (fp32)
//   out[t, :] = sum_j y[route_to_send[t k + j], :]     (fp32, slot order)
//
// Routing tables and tile lists are those of the bf16 layer. The experts' outputs
// stay in fp32 until the slots are summed: in bf16 each would be off by as much
// as the result is by its own rounding.
#include "fp8_tile.h"

namespace {

struct LayerArgs {
  const uint8_t* x;     // rows [., K]
  const uint8_t* xs;    // their scales [., K / 128]
  const int32_t* rows;  // row of x of expert-major row i, or NULL: i
  const uint8_t* w;     // [E, C, K]
  const uint8_t* ws;    // [E, C / 128, K / 128]
  const float* weight;  // routing weight of row i (FC1)
  void* out;            // E4M3 [R, I] (FC1) or fp32 [R, C]
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

// ------------------------------------------------------------------ few rows an expert
// An expert's rows against 128 columns of the activation (FC1: 8 waves, each 16
// gate and the 16 up channels of the same columns) or 32 W channels (FC2).
// Weights and rows go straight from memory into the matrix instruction: weights
// are its rows, 16 NT tokens at a time its columns. Every wave sums the whole
// of K, U blocks in flight.
template <bool FC1, int NT, int W, int U>
__global__ __launch_bounds__(W * 64) void fp8_stream_kernel(LayerArgs p) {
  static_assert(W == (FC1 ? 8 : 4), "a workgroup has 128 columns");
  __shared__ uint32_t tops[FC1 ? W : 1][NT * 16];
  const int cblocks = FC1 ? p.inter / kBlock : p.c / (32 * W);
  const int tile = blockIdx.x / cblocks, cb = blockIdx.x % cblocks;
  if (tile >= p.tl->count) return;
  const int4 t = p.tl->tiles[tile];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), j = lane & 15, q = lane >> 4;
  const int kb = p.k / kBlock;
  // the wave's first channel in either group of 16
  const int c0 = FC1 ? cb * kBlock + wave * 16 : (cb * W + wave) * 32;
  const int c1 = FC1 ? p.inter + c0 : c0 + 16;
  const uint8_t* const w = p.w + static_cast<int64_t>(t.x) * p.c * p.k;
  const uint8_t* const ws = p.ws + static_cast<int64_t>(t.x) * (p.c / kBlock) * kb;
  const uint8_t* const w0 = w + static_cast<int64_t>(c0 + j) * p.k + 16 * q;
  const uint8_t* const w1 = w + static_cast<int64_t>(c1 + j) * p.k + 16 * q;
  const uint8_t* const s0 = ws + static_cast<int64_t>(c0 / kBlock) * kb;
  const uint8_t* const s1 = ws + static_cast<int64_t>(c1 / kBlock) * kb;
  for (int r = t.y; r < t.z; r += NT * 16) {
    const uint8_t* x[NT];
    const uint8_t* xs[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int i = min(r + n * 16 + j, t.z - 1);
      const int64_t row = p.rows ? p.rows[i] : i;
      x[n] = p.x + row * p.k + 16 * q;
      xs[n] = p.xs + row * kb;
    }
    f32x4 acc[2][NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) acc[0][n] = acc[1][n] = f32x4{0, 0, 0, 0};
    auto steps = [&](auto count, int b) {
      constexpr int N = decltype(count)::value;
      i32x8 wv[N][2], xv[N][NT];
      uint32_t sv[N][2], sx[N][NT];
#pragma unroll
      for (int u = 0; u < N; ++u) {
        const int at = (b + u) * kBlock;
        wv[u][0] = load32(w0 + at);
        wv[u][1] = load32(w1 + at);
        sv[u][0] = s0[b + u];
        sv[u][1] = s1[b + u];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          xv[u][n] = load32(x[n] + at);
          sx[u][n] = xs[n][b + u];
        }
      }
#pragma unroll
      for (int u = 0; u < N; ++u)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int g = 0; g < 2; ++g) acc[g][n] = Op16::mac(wv[u][g], xv[u][n], acc[g][n], sv[u][g], sx[u][n]);
    };
    int b = 0;
    for (; b + U <= kb; b += U) steps(std::integral_constant<int, U>{}, b);
    for (; b < kb; ++b) steps(std::integral_constant<int, 1>{}, b);

    if constexpr (FC1) {
      float act[NT][4];
      __syncthreads();  // the chunk before has read `tops`
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const float weight = p.weight[min(r + n * 16 + j, t.z - 1)];
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          act[n][i] = gated_act(p.act_kind, acc[0][n][i], acc[1][n][i], p.beta, p.lbeta, p.limit) * weight;
          top = max(top, abs_bits(act[n][i]));
        }
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
        if (q == 0) tops[wave][n * 16 + j] = top;
      }
      __syncthreads();
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int i = r + n * 16 + j;
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < W; ++k) top = max(top, tops[k][n * 16 + j]);
        const BlockScale s(top);
        if (i >= t.z) continue;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + static_cast<int64_t>(i) * p.inter + c0 + 4 * q) =
            s.pack4(act[n][0], act[n][1], act[n][2], act[n][3]);
        if (wave == 0 && q == 0) p.out_scale[static_cast<int64_t>(i) * (p.inter / kBlock) + cb] = static_cast<uint8_t>(s.byte);
      }
    } else {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int i = r + n * 16 + j;
        if (i >= t.z) continue;
#pragma unroll
        for (int g = 0; g < 2; ++g)
          *reinterpret_cast<f32x4*>(static_cast<float*>(p.out) + static_cast<int64_t>(i) * p.c + c0 + g * 16 + 4 * q) = acc[g][n];
      }
    }
  }
}

// ------------------------------------------------------------------ many rows an expert
// Rows of K bytes, K a multiple of 128: 16-byte vectors of a stage, NT threads.
template <int ROWS, int NT>
struct RowPanel {
  // 32 rows of 8 waves: the upper half of the threads has a vector that the lower one has too
  static constexpr int PER = (ROWS * 8 + NT - 1) / NT;
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
      const int c = (v * NT + threadIdx.x) % (ROWS * 8);
      off[v] = static_cast<uint32_t>(row(c / 8)) * static_cast<uint32_t>(K) + c % 8 * 16;
    }
  }
  __device__ __forceinline__ void load_one(Stage& r, int v, int k) const {
    load_at(r.d[v], base + k, off[v]);
  }
  __device__ __forceinline__ void put_one(int8_t* lds, const Stage& r, int v) const {
    const int c = (v * NT + threadIdx.x) % (ROWS * 8);
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

// One tile of 16 MI WM rows of an expert by 256 channels: with FC1 128 columns
// of the activation, a wave's channels gate and up of the same columns.
template <bool FC1, int MI, int WM, int WN, int PRE>
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
  tile_sums<Op16, BM, BN, WM, WN, 1, PRE, FC1 ? 2 : 1>(smem, pa, pb, p.k, sa, sb, acc);
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

// A tile list's tile and a run of 256 channels (128 columns of the activation)
// a workgroup. Tile m runs on XCD m % 8 with all its channels, so that its rows
// come from one L2. The instructions fit the tile's rows: tiles of experts with
// fewer do not multiply what is not there.
template <bool FC1, int ROWS>
__global__ __launch_bounds__(512) void fp8_rows_kernel(LayerArgs p) {
  __shared__ __attribute__((aligned(1024))) int8_t lds[2 * (ROWS + 256) * BK];
  const int cblocks = FC1 ? p.inter / kBlock : (p.c + 255) / 256;
  const int slot = blockIdx.x >> 3, tile = slot / cblocks * 8 + (blockIdx.x & 7), cb = slot % cblocks;
  if (tile >= p.tl->count) return;
  const int4 t = p.tl->tiles[tile];
  const int rows = t.z - t.y;
  if constexpr (ROWS == kStreamRows) {
    if (rows <= 32) return rows_tile<FC1, 1, 2, 4, 1>(p, lds, t, cb);
    if (rows <= 64) return rows_tile<FC1, 2, 2, 4, 1>(p, lds, t, cb);
    if (rows <= 96) return rows_tile<FC1, 3, 2, 4, 1>(p, lds, t, cb);
    if (rows <= 128) return rows_tile<FC1, 4, 2, 4, 1>(p, lds, t, cb);
    rows_tile<FC1, 5, 2, 4, 1>(p, lds, t, cb);
  } else {
    if (rows <= 128) return rows_tile<FC1, 2, 4, 2, 1>(p, lds, t, cb);
    rows_tile<FC1, 4, 4, 2, 1>(p, lds, t, cb);
  }
}

// out[t, :] = sum of the token's slots in slot order; a thread has 8 columns.
__global__ __launch_bounds__(256) void fp8_combine_kernel(const float* y, const int32_t* route_to_send, int64_t tokens,
                                                          int32_t top_k, int32_t hidden, uint16_t* out) {
  const int chunks = hidden / 8;
  const int64_t total = tokens * chunks;
  for (int64_t v = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; v < total; v += static_cast<int64_t>(gridDim.x) * 256) {
    const int64_t token = v / chunks;
    const int c = static_cast<int>(v - token * chunks) * 8;
    float sum[8] = {};
    for (int j = 0; j < top_k; ++j) {
      const int32_t row = route_to_send[token * top_k + j];
      if (row < 0) continue;
      const f32x4* from = reinterpret_cast<const f32x4*>(y + static_cast<int64_t>(row) * hidden + c);
      const f32x4 a = from[0], b = from[1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sum[i] += a[i];
        sum[4 + i] += b[i];
      }
    }
    *reinterpret_cast<uint4*>(out + token * hidden + c) =
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

struct Scratch {
  int32_t *counts, *offsets, *send_route, *send_token, *route_to_send;
  float* weight_perm;
  void *tiles, *route_ws;
  uint8_t *act, *act_scale;
  float* y;
  size_t tiles_bytes, route_ws_bytes, bytes;

  Scratch(void* base, int64_t R, int E, int hidden, int inter) {
    Carver c{static_cast<char*>(base)};
    const size_t r = static_cast<size_t>(R);
    tiles_bytes = mm_tile_lists_bytes(R, E);
    route_ws_bytes = mm_route_workspace_bytes(R, E);
    y = c.take<float>(r * hidden * 4);
    act = c.take<uint8_t>(r * inter);
    act_scale = c.take<uint8_t>(r * (inter / kBlock));
    route_ws = c.take<void>(route_ws_bytes);
    tiles = c.take<void>(tiles_bytes);
    counts = c.take<int32_t>(static_cast<size_t>(E) * 4);
    offsets = c.take<int32_t>(static_cast<size_t>(E + 1) * 4);
    send_route = c.take<int32_t>(r * 4);
    send_token = c.take<int32_t>(r * 4);
    route_to_send = c.take<int32_t>(r * 4);
    weight_perm = c.take<float>(r * 4);
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

int launch(void (*kernel)(LayerArgs), int64_t blocks, int threads, const LayerArgs& p, hipStream_t s) {
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
  MM_CHECK_ARG(((reinterpret_cast<uintptr_t>(scratch) | reinterpret_cast<uintptr_t>(out)) & 15) == 0,
               "mm_moe_fp8: scratch and out must be 16-byte aligned");
  if (!scratch || scratch_bytes < s.bytes) {
    mm_set_error("mm_moe_fp8: scratch needs %zu bytes", s.bytes);
    return MM_E_WS;
  }
  int rc = mm_route_tiles(selected, R, top_k, E, routing_weights, s.counts, s.offsets, s.send_route, s.send_token,
                          s.route_to_send, s.weight_perm, s.tiles, s.tiles_bytes, s.route_ws, s.route_ws_bytes, stream);
  if (rc) return rc;
  const hipStream_t hs = mm_hip_stream(stream);
  // rows an expert on average
  const int64_t mean = (R + E - 1) / E;
  const int height = mean > kStreamRows ? 256 : kStreamRows;
  const TileList* tl = mm_tile_list_of(s.tiles, R, E, height);
  const int64_t tiles = mm_max_m_tiles(R, E, height), tiles8 = (tiles + 7) / 8 * 8;
  const LayerArgs fc1{x, x_scale, s.send_token, w1, w1_scale, s.weight_perm, s.act, s.act_scale, tl, hidden, 2 * inter, inter,
                      act_kind, situ_beta, situ_linear_beta, clamp_limit};
  const LayerArgs fc2{s.act, s.act_scale, nullptr, w2, w2_scale, nullptr, s.y, nullptr, tl, inter, hidden, inter, 0, 0, 0, 0};
  if (mean <= 16) {
    rc = launch(fp8_stream_kernel<true, 1, 8, 2>, tiles * (inter / kBlock), 512, fc1, hs);
    if (!rc) rc = launch(fp8_stream_kernel<false, 1, 4, 2>, tiles * (hidden / kBlock), 256, fc2, hs);
  } else {
    rc = launch(height == 256 ? fp8_rows_kernel<true, 256> : fp8_rows_kernel<true, kStreamRows>, tiles8 * (inter / kBlock),
                512, fc1, hs);
    if (!rc)
      rc = launch(height == 256 ? fp8_rows_kernel<false, 256> : fp8_rows_kernel<false, kStreamRows>,
                  tiles8 * ((hidden + 255) / 256), 512, fc2, hs);
  }
  if (rc) return rc;
  const int64_t groups = (tokens * (hidden / 8) + 255) / 256;
  fp8_combine_kernel<<<static_cast<uint32_t>(groups < 65536 ? groups : 65536), 256, 0, hs>>>(s.y, s.route_to_send, tokens, top_k,
                                                                                             hidden, out);
  return mm_check_launch("fp8_combine_kernel");
}
