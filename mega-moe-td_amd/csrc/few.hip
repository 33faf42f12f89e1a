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
// result column depends on its own token only. A pass takes 16, 32 or 64 rows of
// an expert; the weights of a further pass come from L2. The waves of
// a workgroup share the sum's axis and join through LDS in wave order. The
// second launch leaves fp32 rows in scratch; the workgroup that finishes a
// tile of columns last adds the tokens' slots in slot order. Every sum has a fixed order.
#include <type_traits>

#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kGroup = MM_FEW_ACT_GROUP;
constexpr float kScaleFloor = 1e-30f;
// 32-bit byte offsets of a lane: 24 rows of w1 (4 I bytes each), 64 tokens of x
// (2 H), and the activation's routes (checked with the sizes)
constexpr int kMaxDim = 1 << 20;
constexpr int64_t kMaxStride = int64_t(1) << 25;  // and 24 rows of w2
constexpr int kMaxInt8Hidden = (1 << 17) - 1;      // an int32 sum of products of -128 and -128

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
  int32_t* done;              // [fc2_tiles + 1]: arrivals at each tile, then the distinct experts
  bf16* out;                  // [T, H]
  int32_t slots;              // experts or routes, each with all column tiles
  int32_t tiles, fc2_tiles;   // column tiles of this launch, and of the second
};

// Workgroup ids go round the 8 XCDs. Eight neighbouring tiles run on one XCD,
// at about the same time: narrow ones share lines, and an expert's rows are
// read in runs of a kilobyte.
constexpr int kNear = 8;
__device__ __forceinline__ int near_block(int blocks) {
  constexpr int G = 8 * kNear;
  const int b = blockIdx.x, base = b / G * G;
  if (base + G > blocks) return b;
  return base + (b & 7) * kNear + (b - base) / 8;
}

// What a workgroup works on. A slot of the grid is an expert where the experts
// are no more than the routes, else a route, of which the first with its expert
// does the work. `list` (R entries) gets the routes of the slot's expert in
// ascending order, `valid` a bit for every route with an expert; count is 0 if
// the slot has no work. Every wave scans for itself and writes the same values
// to LDS: no barrier.
struct Work {
  int slot, tile, expert, count;
  __device__ __forceinline__ Work(const FewArgs& p, uint16_t* list, uint64_t* valid) {
    const int block = near_block(p.slots * p.tiles), lane = threadIdx.x & 63;
    slot = block / p.tiles;
    tile = block % p.tiles;
    count = 0;
    const bool by_expert = p.E <= p.R;
    expert = by_expert ? slot : __builtin_amdgcn_readfirstlane(p.selected[slot]);
    if (static_cast<uint32_t>(expert) >= static_cast<uint32_t>(p.E)) return;
    int n = 0, first = slot;
    for (int base = 0; base < p.R; base += 256) {
      int e[4];  // loaded together
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = base + u * 64 + lane;
        e[u] = r < p.R ? p.selected[r] : -1;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r0 = base + u * 64;
        if (r0 >= p.R) break;
        const uint64_t mask = __ballot(e[u] == expert);
        const uint64_t live = __ballot(static_cast<uint32_t>(e[u]) < static_cast<uint32_t>(p.E));
        if (n == 0 && mask) first = r0 + __ffsll(static_cast<unsigned long long>(mask)) - 1;
        if (e[u] == expert) list[n + __popcll(mask & ((1ull << lane) - 1))] = static_cast<uint16_t>(r0 + lane);
        if (lane == 0) valid[r0 >> 6] = live;
        n += __popcll(mask);
      }
    }
    if (by_expert || first == slot) count = n;
  }
};

// Clears the second launch's arrival counters and counts the distinct experts,
// each of which arrives once at every tile.
template <int THREADS>
__device__ void prepare_done(const FewArgs& p, uint32_t* bits) {
  for (int i = threadIdx.x; i < p.fc2_tiles; i += THREADS) p.done[i] = 0;
  const int words = (p.E + 31) / 32;
  for (int i = threadIdx.x; i < words; i += THREADS) bits[i] = 0;
  __syncthreads();
  for (int r = threadIdx.x; r < p.R; r += THREADS) {
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
}

// ------------------------------------------------------------------ products
// Every operand is addressed as a uniform base and a 32-bit offset of the lane.
// A step's loads are issued together and awaited by its own multiplication:
// what keeps the memory busy is that two to five workgroups fit a CU. A second
// and a third step in registers cost that and were slower (8 experts' weights
// are 10% faster with them, 112 experts' 10 to 20% slower).

// Weights with their columns contiguous, CL columns a lane: 8 rows of CL
// columns are transposed in registers (4 v_perm for each 16 bytes) into CL
// operands of 16 columns x 32 rows. Column of operand c, row i: CL * i + c.
// w_off: the lane's columns in row 8 * (lane / 16). Lines that a wave reads
// whole carry the non-temporal hint (7168 x 4096, 64-column tiles: 373 us
// against 411 for 41 experts); halves of lines do not, as the hint drops the
// half that the neighbour comes for (640 against 503).
template <int CL, int NT, bool STREAM>
struct ColumnStep {
  typedef uint32_t Raw __attribute__((ext_vector_type(CL / 2)));
  Raw w[8];
  bf16x8 x[NT];
  __device__ __forceinline__ void load(const char* wp, uint32_t w_off, int64_t row_bytes, const char* xp,
                                       const uint32_t (&x_off)[NT]) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const Raw* p = reinterpret_cast<const Raw*>(wp + r * row_bytes + w_off);
      w[r] = STREAM ? __builtin_nontemporal_load(p) : *p;
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) __builtin_memcpy(&x[n], xp + x_off[n], 16);
  }
  __device__ __forceinline__ void multiply(f32x4 (&acc)[CL * NT]) const {
#pragma unroll
    for (int c = 0; c < CL; ++c) {
      const uint32_t sel = (c & 1) ? 0x07060302u : 0x05040100u;
      u32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_perm(w[2 * i + 1][c >> 1], w[2 * i][c >> 1], sel);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        acc[c * NT + n] =
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v), x[n], acc[c * NT + n], 0, 0, 0);
    }
  }
};

// Weights with the sum's axis contiguous: 16 bytes a lane are an operand as
// they are, 16 weight rows and 64 bytes of the sum's axis an instruction. A
// piece is 128 bytes, so that a wave asks for both halves of a line, one after
// the other (41 experts of 4096 x 7168 in int8: 205 us, in pieces of 64 bytes
// 236), without the non-temporal hint, which drops the second half (244).
// w[g][h]: half h of group g.
template <int G>
struct RowStep {
  i32x4 w[G][2];
  __device__ __forceinline__ void load(const char* wp, int64_t group_bytes, uint32_t w_off) {
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int h = 0; h < 2; ++h) __builtin_memcpy(&w[g][h], wp + g * group_bytes + h * 64 + w_off, 16);
  }
};
// The tokens' two operands of a piece.
template <int NT>
struct TokenStep {
  i32x4 x[NT][2];
  __device__ __forceinline__ void load(const char* xp, const uint32_t (&x_off)[NT]) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) __builtin_memcpy(&x[n][h], xp + h * 64 + x_off[n], 16);
  }
};

// The routes of the lane's columns: NT blocks of 16, the last route repeated.
template <int NT>
__device__ __forceinline__ void routes_of(const uint16_t* list, int c0, int count, int (&route)[NT]) {
#pragma unroll
  for (int n = 0; n < NT; ++n) route[n] = list[min(c0 + n * 16 + static_cast<int>(threadIdx.x & 15), count - 1)];
}

template <int N, class V>
__device__ __forceinline__ void clear(V (&acc)[N]) {
#pragma unroll
  for (int a = 0; a < N; ++a) acc[a] = V{0, 0, 0, 0};
}

// The W waves of a workgroup share the sum's axis: of n pieces, wave w takes w,
// w + W, ... Their partial sums are joined through LDS in the order of the waves.
template <int W>
struct Waves {
  int wave;
  __device__ __forceinline__ Waves() : wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {}
  template <int N, class V>
  __device__ __forceinline__ void leave(V* red, const V (&acc)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) red[(wave * N + i) * 64 + (threadIdx.x & 63)] = acc[i];
  }
  // operand `op` of the lane
  template <int N, class V>
  __device__ __forceinline__ V join(const V* red, int op) const {
    const V* r = red + op * 64 + (threadIdx.x & 63);
    V s = r[0];
#pragma unroll
    for (int k = 1; k < W; ++k) s += r[k * N * 64];
    return s;
  }
};

// LDS of a launch beside its fixed arrays: `valid`, then `list`.
extern __shared__ uint64_t route_lds[];
__device__ __forceinline__ uint16_t* list_of(const FewArgs& p) {
  return reinterpret_cast<uint16_t*>(route_lds + (p.R + 63) / 64);
}
size_t route_lds_bytes(int R) { return static_cast<size_t>((R + 63) / 64) * 8 + static_cast<size_t>(R) * 2; }

// ------------------------------------------------------------------ first launch, bf16
// Tile of C = 8 * CL columns: operand rows 0..7 are gate, 8..15 up columns.
template <int CL, int W, int NT>
__global__ __launch_bounds__(W * 64) void few_fc1_kernel(FewArgs p) {
  constexpr int C = 8 * CL;
  __shared__ f32x4 red[W * CL * NT * 64];
  __shared__ __attribute__((aligned(16))) bf16 stage[NT * 16][C + 8];
  const Waves<W> ws;
  const int tid = threadIdx.x, lane = tid & 63, j = lane & 15, q = lane >> 4;
  uint16_t* list = list_of(p);
  if (static_cast<int>(blockIdx.x) == p.slots * p.tiles) {  // the workgroup behind the tiles
    prepare_done<W * 64>(p, reinterpret_cast<uint32_t*>(red));
    return;
  }
  const Work wk(p, list, route_lds);
  if (!wk.count) return;
  const int64_t row_bytes = 4 * static_cast<int64_t>(p.I);
  const char* w = static_cast<const char*>(p.w1) + static_cast<int64_t>(wk.expert) * p.H * row_bytes + wk.tile * C * 2;
  const uint32_t w_off = static_cast<uint32_t>(8 * q * row_bytes) + (j < 8 ? 0 : 2 * p.I) + CL * 2 * (j & 7);
  for (int c0 = 0; c0 < wk.count; c0 += NT * 16) {
    int route[NT];
    uint32_t x_off[NT];
    float wt[NT];
    routes_of<NT>(list, c0, wk.count, route);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      x_off[n] = (static_cast<uint32_t>(route[n] / p.top_k) * p.H + 8 * q) * 2;
      wt[n] = p.w[route[n]];
    }
    f32x4 acc[CL * NT];
    clear(acc);
    for (int s = ws.wave; s < p.H / 32; s += W) {
      ColumnStep<CL, NT, C * 2 >= 128> st;
      st.load(w + s * 32 * row_bytes, w_off, row_bytes, static_cast<const char*>(p.x) + s * 64, x_off);
      st.multiply(acc);
    }
    ws.leave(red, acc);
    __syncthreads();
    for (int c = ws.wave; c < CL; c += W) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const f32x4 v = ws.template join<CL * NT>(red, c * NT + n);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float up = __shfl(v[r], (lane + 32) & 63);
          if (lane < 32)
            stage[n * 16 + j][CL * (4 * q + r) + c] =
                static_cast<bf16>(gated_act(p.act_kind, v[r], up, p.beta, p.lbeta, p.limit) * wt[n]);
        }
      }
    }
    __syncthreads();
    for (int item = tid; item < NT * 16 * (C / 8); item += W * 64) {
      const int row = item / (C / 8), vec = item % (C / 8);
      if (c0 + row < wk.count)
        *reinterpret_cast<uint4*>(static_cast<bf16*>(p.act) + static_cast<int64_t>(list[c0 + row]) * p.I + wk.tile * C +
                                  vec * 8) = *reinterpret_cast<const uint4*>(&stage[row][vec * 8]);
    }
  }
}

// ------------------------------------------------------------------ second launch
// y crosses the XCDs' L2 caches inside the launch: it is written and read with
// agent-scope accesses, which go past them. A release fence would write back
// the whole L2 of the XCD for every workgroup (8 experts, 2048 columns: 41 us
// against 10). What orders the hand-over instead: an agent-scope store writes
// through to memory and counts as outstanding (vmcnt) until it is there; a wave
// waits for its own, the barrier for the workgroup's waves, and only then does
// the workgroup arrive. The last to arrive reads y behind that, and no cache of
// its XCD can hold an older copy of a line: within the launch nobody has read y,
// and a route's columns of a tile, whole lines, are written by one workgroup.
__device__ __forceinline__ void put_y(float* p, const f32x4& v) {
  const uint64_t* w = reinterpret_cast<const uint64_t*>(&v);
  uint64_t* d = reinterpret_cast<uint64_t*>(p);
  __hip_atomic_store(d, w[0], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store(d + 1, w[1], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Called by every workgroup with work once its part of y is written; the last
// of the tile adds the tokens' slots. y holds the tile's C columns in the order
// that column_of gives. A thread adds 4 columns of ITEMS tokens with all loads
// of 8 slots in flight.
template <int C, int THREADS, class ColumnOf>
__device__ __forceinline__ void finish(const FewArgs& p, const Work& wk, int live, ColumnOf column_of) {
  constexpr int ITEMS = 2, Q = C / 4;
  __shared__ int last;
  // each wave's stores have reached memory before its workgroup arrives
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(&p.done[wk.tile], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == live - 1;
  __syncthreads();
  if (!last) return;
  const int col0 = wk.tile * C, items = p.tokens * Q;
  for (int i0 = threadIdx.x; i0 < items; i0 += ITEMS * THREADS) {
    f32x4 s[ITEMS];
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) s[u] = f32x4{0, 0, 0, 0};
    for (int k0 = 0; k0 < p.top_k; k0 += 8) {
      uint64_t v[ITEMS][8][2];
#pragma unroll
      for (int u = 0; u < ITEMS; ++u) {
        const int i = i0 + u * THREADS;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int r = i / Q * p.top_k + k0 + k;
          v[u][k][0] = v[u][k][1] = 0;
          if (i < items && k0 + k < p.top_k && ((route_lds[r >> 6] >> (r & 63)) & 1)) {
            const uint64_t* y = reinterpret_cast<const uint64_t*>(p.y + static_cast<int64_t>(r) * p.H + col0 + i % Q * 4);
            v[u][k][0] = __hip_atomic_load(y, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            v[u][k][1] = __hip_atomic_load(y + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < ITEMS; ++u)
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[u][r] += __uint_as_float(static_cast<uint32_t>(v[u][k][r >> 1] >> (32 * (r & 1))));
    }
#pragma unroll
    for (int u = 0; u < ITEMS; ++u) {
      const int i = i0 + u * THREADS;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (i < items) p.out[static_cast<int64_t>(i / Q) * p.H + col0 + column_of(i % Q * 4 + r)] = static_cast<bf16>(s[u][r]);
    }
  }
}

// No route has an expert: the first slot's workgroups write the empty sums.
template <int C, int THREADS>
__device__ __forceinline__ void finish_empty(const FewArgs& p, const Work& wk) {
  for (int i = threadIdx.x; i < p.tokens * C; i += THREADS)
    p.out[static_cast<int64_t>(i / C) * p.H + wk.tile * C + i % C] = static_cast<bf16>(0.0f);
}

// ROWS: w2's sum axis is contiguous (N groups of 16 columns), else its columns
// are (N = CL columns a lane).
template <bool ROWS, int N, int W, int NT>
__global__ __launch_bounds__(W * 64) void few_fc2_kernel(FewArgs p) {
  constexpr int C = 16 * N;
  __shared__ f32x4 red[W * N * NT * 64];
  const Waves<W> ws;
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  uint16_t* list = list_of(p);
  const Work wk(p, list, route_lds);
  const int live = p.done[p.tiles];
  if (live == 0 && wk.slot == 0) finish_empty<C, W * 64>(p, wk);
  if (!wk.count) return;
  const int col = wk.tile * C;
  const int64_t row_bytes = 2 * p.w2_ld;
  const char* w = static_cast<const char*>(p.w2) + 2 * static_cast<int64_t>(wk.expert) * p.w2_se +
                  (ROWS ? col * row_bytes : col * 2);
  const uint32_t w_off = ROWS ? static_cast<uint32_t>(j * row_bytes) + 16 * q
                              : static_cast<uint32_t>(8 * q * row_bytes) + N * 2 * j;
  const char* x = static_cast<const char*>(p.act);
  for (int c0 = 0; c0 < wk.count; c0 += NT * 16) {
    int route[NT];
    uint32_t x_off[NT];
    routes_of<NT>(list, c0, wk.count, route);
#pragma unroll
    for (int n = 0; n < NT; ++n) x_off[n] = (static_cast<uint32_t>(route[n]) * p.I + 8 * q) * 2;
    f32x4 acc[N * NT];
    clear(acc);
    if constexpr (ROWS) {
      for (int s = ws.wave; s < p.I / 64; s += W) {
        RowStep<N> st;
        TokenStep<NT> tok;
        st.load(w + s * 128, 16 * row_bytes, w_off);
        tok.load(x + s * 128, x_off);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int g = 0; g < N; ++g)
#pragma unroll
            for (int n = 0; n < NT; ++n)
              acc[g * NT + n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, st.w[g][h]),
                                                                        __builtin_bit_cast(bf16x8, tok.x[n][h]),
                                                                        acc[g * NT + n], 0, 0, 0);
      }
    } else {
      for (int s = ws.wave; s < p.I / 32; s += W) {
        ColumnStep<N, NT, true> st;
        st.load(w + s * 32 * row_bytes, w_off, row_bytes, x + s * 64, x_off);
        st.multiply(acc);
      }
    }
    if (c0) __syncthreads();  // the tokens before have been joined
    ws.leave(red, acc);
    __syncthreads();
    // rows 4q..4q + 3 of an operand and token j are kept side by side in y
    for (int op = ws.wave; op < N * NT; op += W) {
      const f32x4 v = ws.template join<N * NT>(red, op);
      const int at = c0 + op % NT * 16 + j;
      if (at < wk.count) put_y(p.y + static_cast<int64_t>(list[at]) * p.H + col + op / NT * 16 + 4 * q, v);
    }
  }
  finish<C, W * 64>(p, wk, live, [](int at) { return ROWS ? at : at % 16 * N + at / 16; });
}

// ------------------------------------------------------------------ int8
// Tile of 32 columns: operands 0, 1 are gate rows of w1, 2, 3 up rows. The
// wave that joins 16 tokens has their 32 columns in its registers, 8 of a token
// in a lane, the others 16, 32 and 48 lanes on.
template <int W, int NT>
__global__ __launch_bounds__(W * 64) void few_fc1_int8_kernel(FewArgs p) {
  constexpr int C = kGroup, G = 2;
  __shared__ i32x4 red[W * 2 * G * NT * 64];
  const Waves<W> ws;
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  uint16_t* list = list_of(p);
  if (static_cast<int>(blockIdx.x) == p.slots * p.tiles) {  // the workgroup behind the tiles
    prepare_done<W * 64>(p, reinterpret_cast<uint32_t*>(red));
    return;
  }
  const Work wk(p, list, route_lds);
  if (!wk.count) return;
  const int col = wk.tile * C;
  const int64_t up_bytes = static_cast<int64_t>(p.I) * p.H;
  const char* w = static_cast<const char*>(p.w1) + 2 * wk.expert * up_bytes + static_cast<int64_t>(col) * p.H;
  const uint32_t w_off = j * p.H + 16 * q;
  for (int c0 = 0; c0 < wk.count; c0 += NT * 16) {
    int routes[NT];
    uint32_t x_off[NT];
    routes_of<NT>(list, c0, wk.count, routes);
#pragma unroll
    for (int n = 0; n < NT; ++n) x_off[n] = static_cast<uint32_t>(routes[n] / p.top_k) * p.H + 16 * q;
    i32x4 acc[2 * G * NT];
    clear(acc);
    for (int s = ws.wave; s < p.H / 128; s += W) {
      RowStep<G> gate, up;
      TokenStep<NT> tok;
      gate.load(w + s * 128, 16 * p.H, w_off);
      up.load(w + up_bytes + s * 128, 16 * p.H, w_off);
      tok.load(static_cast<const char*>(p.x) + s * 128, x_off);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            i32x4 &a = acc[g * NT + n], &b = acc[(G + g) * NT + n];
            a = __builtin_amdgcn_mfma_i32_16x16x64_i8(gate.w[g][h], tok.x[n][h], a, 0, 0, 0);
            b = __builtin_amdgcn_mfma_i32_16x16x64_i8(up.w[g][h], tok.x[n][h], b, 0, 0, 0);
          }
    }
    if (c0) __syncthreads();  // the tokens before have been joined
    ws.leave(red, acc);
    __syncthreads();
    // one wave joins a block of 16 tokens
    for (int n = ws.wave; n < NT; n += W) {
      const int at = c0 + n * 16 + j, route = list[min(at, wk.count - 1)];
      // an infinite scale marks a broken row as NaN does; a clamp or a tanh would hide it
      const float mark = p.x_scale[route / p.top_k], wt = p.w[route];
      const float sx = fabsf(mark) < __builtin_inff() ? mark : __uint_as_float(0x7fc00000u);
      const float* sc = p.w1_scale + static_cast<int64_t>(wk.expert) * 2 * p.I + col + 4 * q;
      float a[G][4];
      uint32_t top = 0;  // of the bit patterns, where NaN lies above infinity
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const i32x4 gate = ws.template join<2 * G * NT>(red, g * NT + n);
        const i32x4 up = ws.template join<2 * G * NT>(red, (G + g) * NT + n);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          a[g][r] = gated_act(p.act_kind, static_cast<float>(gate[r]) * (sx * sc[g * 16 + r]),
                              static_cast<float>(up[r]) * (sx * sc[p.I + g * 16 + r]), p.beta, p.lbeta, p.limit) * wt;
          top = max(top, __float_as_uint(a[g][r]) & 0x7fffffffu);
        }
      }
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
      top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
      if (at >= wk.count) continue;
      const bool finite = top < 0x7f800000u;
      const float most = fmaxf(__uint_as_float(top), kScaleFloor), inv = finite ? 127.0f / most : 0.0f;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        uint32_t b = 0;
#pragma unroll
        for (int r = 0; r < 4; ++r)
          b |= static_cast<uint32_t>(finite ? static_cast<int>(__builtin_rintf(a[g][r] * inv)) & 0xff : 0) << (8 * r);
        *reinterpret_cast<uint32_t*>(static_cast<int8_t*>(p.act) + static_cast<int64_t>(route) * p.I + col + g * 16 + 4 * q) = b;
      }
      if (q == 0)
        p.act_scale[static_cast<int64_t>(route) * (p.I / C) + col / C] = finite ? most / 127.0f : __uint_as_float(0x7fc00000u);
    }
  }
}

// Tile of 64 columns. An instruction's 64 elements span two scale groups (the
// operand's lanes 0..31 and 32..63), so each is multiplied with the other's
// activations zeroed and joins the fp32 sum under its own scale.
template <int W, int NT>
__global__ __launch_bounds__(W * 64) void few_fc2_int8_kernel(FewArgs p) {
  constexpr int G = 4, C = 16 * G;
  __shared__ f32x4 red[W * G * NT * 64];
  const Waves<W> ws;
  const int lane = threadIdx.x & 63, j = lane & 15, q = lane >> 4;
  uint16_t* list = list_of(p);
  const Work wk(p, list, route_lds);
  const int live = p.done[p.tiles];
  if (live == 0 && wk.slot == 0) finish_empty<C, W * 64>(p, wk);
  if (!wk.count) return;
  const int col = wk.tile * C;
  const char* w = static_cast<const char*>(p.w2) + (static_cast<int64_t>(wk.expert) * p.H + col) * p.I;
  const uint32_t w_off = j * p.I + 16 * q;
  for (int c0 = 0; c0 < wk.count; c0 += NT * 16) {
    int route[NT];
    uint32_t x_off[NT], sc_off[NT];
    routes_of<NT>(list, c0, wk.count, route);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      x_off[n] = static_cast<uint32_t>(route[n]) * p.I + 16 * q;
      sc_off[n] = static_cast<uint32_t>(route[n]) * (p.I / kGroup) * 4;
    }
    f32x4 acc[G * NT];
    clear(acc);
    for (int s = ws.wave; s < p.I / 128; s += W) {
      RowStep<G> st;
      TokenStep<NT> tok;
      f32x4 sv[NT];
      st.load(w + s * 128, 16 * p.I, w_off);
      tok.load(static_cast<const char*>(p.act) + s * 128, x_off);
#pragma unroll
      for (int n = 0; n < NT; ++n)
        __builtin_memcpy(&sv[n], reinterpret_cast<const char*>(p.act_scale) + s * (128 / kGroup * 4) + sc_off[n], 16);
      const i32x4 zero = {0, 0, 0, 0};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const i32x4 lo = lane < 32 ? tok.x[n][h] : zero, hi = lane < 32 ? zero : tok.x[n][h];
#pragma unroll
          for (int g = 0; g < G; ++g) {
            const i32x4 a = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.w[g][h], lo, zero, 0, 0, 0);
            const i32x4 b = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.w[g][h], hi, zero, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[g * NT + n][r] += static_cast<float>(a[r]) * sv[n][2 * h] + static_cast<float>(b[r]) * sv[n][2 * h + 1];
          }
        }
    }
    if (c0) __syncthreads();  // the tokens before have been joined
    ws.leave(red, acc);
    __syncthreads();
    for (int op = ws.wave; op < G * NT; op += W) {
      f32x4 v = ws.template join<G * NT>(red, op);
      const int at = c0 + op % NT * 16 + j, c = col + op / NT * 16 + 4 * q;
      const float* sc = p.w2_scale + static_cast<int64_t>(wk.expert) * p.H + c;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] *= sc[k];
      if (at < wk.count) put_y(p.y + static_cast<int64_t>(list[at]) * p.H + c, v);
    }
  }
  finish<C, W * 64>(p, wk, live, [](int at) { return at; });
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

bool few_sizes_ok(int64_t tokens, int32_t top_k, int32_t E, int32_t H, int32_t I, bool int8) {
  return tokens >= 0 && tokens <= MM_FEW_MAX_TOKENS && top_k > 0 && top_k <= 64 && E > 0 && E <= 32768 && H > 0 &&
         H % 128 == 0 && I > 0 && I % 128 == 0 && H <= (int8 ? kMaxInt8Hidden : kMaxDim) &&
         I <= kMaxDim && tokens * top_k * I < (int64_t(1) << 31);
}

int slots_of(const FewArgs& p) { return p.E <= p.R ? p.E : p.R; }

// One launch: its waves and its tiles of `width` columns.
struct Launch {
  void (*kernel)(FewArgs);
  int waves, width;
};

int launch_both(FewArgs p, const Launch& a, const Launch& b, hipStream_t s) {
  const int slots = slots_of(p), tiles1 = p.I / a.width, tiles2 = p.H / b.width;
  MM_CHECK_ARG(static_cast<int64_t>(slots) * (tiles1 > tiles2 ? tiles1 : tiles2) + 1 < (int64_t(1) << 23),
               "mm_moe_few: too many tiles");
  const size_t lds = route_lds_bytes(p.R);
  p.slots = slots;
  p.fc2_tiles = tiles2;
  p.tiles = tiles1;
  a.kernel<<<slots * tiles1 + 1, a.waves * 64, lds, s>>>(p);
  const int rc = mm_check_launch("few_fc1_kernel");
  if (rc) return rc;
  p.tiles = tiles2;
  b.kernel<<<slots * tiles2, b.waves * 64, lds, s>>>(p);
  return mm_check_launch("few_fc2_kernel");
}

// Blocks of 16 tokens in a pass over an expert's weights, by the mean rows of an
// expert: more than its rows need cost occupancy (60 experts of 8.5 rows: 85 us
// with one, 95 with two), fewer read the weights again (32 of 16 rows: 234 us
// with one, 150 with two; 8 of 64: 30 us with two, 19 with four).
template <class F>
int by_blocks(const FewArgs& p, F&& f) {
  if (p.tokens <= 16 || p.R <= 10 * p.E) return f(std::integral_constant<int, 1>{});
  if (p.tokens <= 32 || p.R <= 24 * p.E) return f(std::integral_constant<int, 2>{});
  return f(std::integral_constant<int, 4>{});
}

}  // namespace

extern "C" size_t mm_moe_few_scratch_bytes(int64_t tokens, int32_t top_k, int32_t hidden, int32_t inter, int32_t int8) {
  if (!few_sizes_ok(tokens, top_k, 1, hidden, inter, int8 != 0)) return 0;
  return FewScratch(tokens * top_k, hidden, inter, int8 != 0).bytes;
}

extern "C" int mm_moe_few(const uint16_t* x, const int32_t* selected, const float* routing_weights, const uint16_t* w1,
                          const uint16_t* w2, int64_t w2_se, int64_t w2_sh, int64_t w2_sf, int64_t tokens,
                          int32_t top_k, int32_t num_experts, int32_t hidden, int32_t inter, int32_t act_kind,
                          float situ_beta, float situ_linear_beta, float clamp_limit, uint16_t* out, void* scratch,
                          size_t scratch_bytes, mm_stream_t stream) {
  MM_CHECK_ARG(few_sizes_ok(tokens, top_k, num_experts, hidden, inter, false), "mm_moe_few: bad sizes");
  MM_CHECK_ARG(w2_sh == 1 || w2_sf == 1, "mm_moe_few: w2 needs a unit stride along hidden or inter");
  MM_CHECK_ARG(w2_sh >= 0 && w2_sh <= kMaxStride && w2_sf >= 0 && w2_sf <= kMaxStride,
               "mm_moe_few: w2 rows more than 2^25 elements apart");
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
            reinterpret_cast<bf16*>(out), 0, 0, 0};
  const hipStream_t s = mm_hip_stream(stream);
  // 64 columns a tile read whole lines; with fewer workgroups than two to a CU
  // 32 columns, twice as many, win (8 experts of 1024 columns: 25 us against 40;
  // of 768, one token: 12.3 against 17.8; 112 experts of 768: 156 against 117)
  const bool wide = static_cast<int64_t>(slots_of(p)) * (inter / 64) >= 512;
  auto run = [&](auto blocks) {
    constexpr int NT = decltype(blocks)::value;
    Launch fc1{few_fc1_kernel<4, 8, NT>, 8, 32};
    if constexpr (NT < 4) {  // the partial sums of 64 tokens and 64 columns do not fit LDS
      if (wide) fc1 = {few_fc1_kernel<8, 8, NT>, 8, 64};
    }
    return launch_both(p, fc1, rows ? Launch{few_fc2_kernel<true, 4, 8, NT>, 8, 64} : Launch{few_fc2_kernel<false, 4, 8, NT>, 8, 64}, s);
  };
  return by_blocks(p, run);
}

extern "C" int mm_moe_few_int8(const int8_t* x, const float* x_scale, const int32_t* selected,
                               const float* routing_weights, const int8_t* w1, const float* w1_scale, const int8_t* w2,
                               const float* w2_scale, int64_t tokens, int32_t top_k, int32_t num_experts,
                               int32_t hidden, int32_t inter, int32_t act_kind, float situ_beta,
                               float situ_linear_beta, float clamp_limit, uint16_t* out, void* scratch,
                               size_t scratch_bytes, mm_stream_t stream) {
  MM_CHECK_ARG(few_sizes_ok(tokens, top_k, num_experts, hidden, inter, true),
               "mm_moe_few_int8: bad sizes (hidden at most %d)", kMaxInt8Hidden);
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
            reinterpret_cast<int32_t*>(base + f.done), reinterpret_cast<bf16*>(out), 0, 0, 0};
  const hipStream_t s = mm_hip_stream(stream);
  auto run = [&](auto blocks) {
    constexpr int NT = decltype(blocks)::value;
    return launch_both(p, {few_fc1_int8_kernel<4, NT>, 4, kGroup}, {few_fc2_int8_kernel<4, NT>, 4, 64}, s);
  };
  return by_blocks(p, run);
}
