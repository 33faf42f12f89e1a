// What the products of 8-bit rows share: tiles, loads of rows at any alignment,
// stages in LDS and the way of results to memory.
#pragma once

#include <type_traits>

#include "common.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
// What results are stored in, at any alignment of their type. One value, not
// elements: the compiler breaks an array's copy up to share it with the branch
// for a row's end (4096 x 256 x 4096: 24 us, 18 so).
typedef int Out4 __attribute__((ext_vector_type(4), aligned(2)));
typedef int Out2 __attribute__((ext_vector_type(2), aligned(2)));

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

// Address of a row as an aligned base and what is left of it. The base is the
// pointer less the rest, not a number made a pointer again, whose loads the
// compiler cannot tell from LDS (it then waits for both kinds at once).
__device__ __forceinline__ const char* aligned_base(const void* p, uint32_t& rest) {
  rest = reinterpret_cast<uintptr_t>(p) & 3;
  return static_cast<const char*>(p) - rest;
}

// Sixteen bytes at a base that is the same for the wave plus a lane's offset. The
// empty instruction keeps the offset's extension to 64 bits in place: in front
// of a loop it is kept there in two registers and the sum is made of vector adds.
template <class T>
__device__ __forceinline__ void load_at(T& to, const char* base, uint32_t off) {
  asm volatile("" : "+v"(off));
  __builtin_memcpy(&to, base + off, 16);
}

// ------------------------------------------------------------------ stages in LDS
constexpr int BK = 128;

// LDS rows of 128 bytes: 16-byte slot s of row r sits at s ^ ((r >> 1) & 7),
// which gives the 16 rows of one pass of a fragment read distinct banks.
__device__ __forceinline__ int slot_of(int r, int s) { return r * BK + ((s ^ ((r >> 1) & 7)) << 4); }

// ROWS rows of a stage: KS sub-panels of [ROWS][128], filled by NT threads. With
// SHIFT a vector's fifth word is the first of the next lane's vector; only the
// last lane of a run loads it, and words are joined on their way to LDS (128 x
// 7169 x 4096 in 32 x 64 tiles: 21 us, 23 with five words loaded by every lane).
// PIN: load_at's loads.
template <int ROWS, int NT, int KS, bool SHIFT, bool PIN = false>
struct Panel {
  static constexpr int VPR = 8 * KS, PER = ROWS * VPR / NT;  // 16-byte vectors a row, a thread
  static_assert(PER * NT == ROWS * VPR && NT % VPR == 0, "whole vectors");
  static constexpr bool CUTS = true;  // has put_cut
  // A run: consecutive lanes with consecutive vectors of a row, within the 16
  // lanes that exchange words.
  static constexpr int LAST = VPR < 16 ? VPR - 1 : 15;
  struct Stage {
    uint32_t d[PER][SHIFT ? 5 : 4];
  };
  const char* base;
  uint32_t off[PER];
  __device__ __forceinline__ void init(const void* p, int64_t ld, int r0, int rows) {
    uint32_t rest;
    base = aligned_base(static_cast<const char*>(p) + r0 * ld, rest);
#pragma unroll
    for (int v = 0; v < PER; ++v) {
      const int c = v * NT + threadIdx.x;
      off[v] = static_cast<uint32_t>(min(c / VPR, rows - 1 - r0)) * static_cast<uint32_t>(ld) + rest + c % VPR * 16;
    }
  }
  __device__ __forceinline__ static bool last_of_run() { return (threadIdx.x & LAST) == LAST; }
  __device__ __forceinline__ void load(Stage& r, int k) const {
#pragma unroll
    for (int v = 0; v < PER; ++v) load_one(r, v, k);
  }
  __device__ __forceinline__ void load_one(Stage& r, int v, int k) const {
    if constexpr (SHIFT) {
      const uint32_t sh = off[v] & 3;
      const char* p = base + k + (off[v] - sh);
      __builtin_memcpy(r.d[v], __builtin_assume_aligned(p, 4), 16);
      if (last_of_run()) __builtin_memcpy(r.d[v] + 4, __builtin_assume_aligned(p + (sh ? 16 : 12), 4), 4);
    } else {
      if constexpr (PIN)
        load_at(r.d[v], base + k, off[v]);
      else
        __builtin_memcpy(r.d[v], base + k + off[v], 16);
    }
  }
  __device__ __forceinline__ void put(int8_t* lds, const Stage& r) const {
#pragma unroll
    for (int v = 0; v < PER; ++v) put_one(lds, r, v);
  }
  __device__ __forceinline__ void put_one(int8_t* lds, const Stage& r, int v) const {
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

// ROWS staged rows of a wave to memory, 16 bytes a lane.
template <int ROWS, int COLS, int PITCH, class T, class Args>
__device__ __forceinline__ void store_rows(const Args& p, const int8_t* staged, int row0, int col0) {
  constexpr int PER = 16 / sizeof(T), LANES = COLS / PER;  // columns a lane, lanes a row
  const int lane = threadIdx.x & 63, r0 = lane / LANES, c = lane % LANES * PER, left = p.n - col0 - c;
  T* out = static_cast<T*>(p.out) + (row0 + r0) * p.ldo + col0 + c;
  const int64_t step = 64 / LANES * p.ldo;
#pragma unroll
  for (int r = 0; r < ROWS; r += 64 / LANES, out += step) {
    if (row0 + r0 + r >= p.m) break;
    const int8_t* from = staged + (r0 + r) * PITCH + c * sizeof(T);
    if (left >= PER) {
      *reinterpret_cast<Out4*>(out) = *reinterpret_cast<const i32x4*>(from);
    } else {
      for (int u = 0; u < left; ++u) out[u] = reinterpret_cast<const T*>(from)[u];
    }
  }
}

}  // namespace
