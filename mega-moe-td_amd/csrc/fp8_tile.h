// The matrix instructions on E4M3 blocks, and tiles of sums through LDS.
//
// Channels (weights) are the rows of an instruction and tokens its columns, so a
// lane holds consecutive channels of one token. A lane's bytes of a block may be
// any of it as long as both operands agree: they are runs of 16.
//
// What the E4M3 instructions sum in: of 8 neighbouring products each is cut 13
// bits below the largest before they are added (measured: with products of 2^p
// and 2^q in one such group the smaller is lost from p - q = 14 on, in another
// group at 24; the same in all three E4M3 instructions). A sum is off by at most
// 7 * 2^-13 (8.5e-4) of its groups' largest products, by 1.4e-5 of it (root mean
// square, no bias) where values are random, whatever its length. Results in 16 bits
// are summed so by choice: of random values it is little beside their own rounding
// (half a step is 2^-8 or 2^-11), the operands were rounded by up to 2^-4, and sums
// in fp32 take twice the matrix time. It shows where large products cancel (448 *
// 448 - 448 * 448 + 1 is 0), and in fp16 where most of a sum lies in products 2^-13
// of their neighbour's size. Results in 32 bits are summed by the bf16 instruction,
// which holds E4M3 values exactly and adds in fp32, at half the rate.
#pragma once

#include "fp8.h"
#include "rows8.h"

namespace {

__device__ __forceinline__ i32x8 join32(const i32x4& lo, const i32x4& hi) {
  return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
}

// 16 x 16 sums over a block of 128 values with the scale byte of the lane's row
// (bits 0-7 of sb, sa): a result is 4 channels from channel(lane) on of the lane's
// token. (32 x 32 x 64 instructions move half as many operand bytes and twice as
// many sums; on registers alone, random values, they reach 3460 TFLOP/s and
// these 3900: the chip is bound by power.)
constexpr int kTile = 16;
__device__ __forceinline__ int token_of(int lane) { return lane & 15; }
__device__ __forceinline__ int channel_of(int lane) { return (lane >> 4) * 4; }

struct Op16 {
  static constexpr int WAVES = 1;  // of a SIMD, at least
  using Frag = i32x8;
  __device__ __forceinline__ static Frag frag(const i32x8& bytes) { return bytes; }
  __device__ __forceinline__ static f32x4 mac(const Frag& b, const Frag& a, const f32x4& c, uint32_t sb, uint32_t sa) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c, 0, 0, 0, static_cast<int>(sb), 0, static_cast<int>(sa));
  }
};

// Op16 with sums in fp32: values in bf16, a block's sum times its power of two.
struct Op16Wide {
  static constexpr int WAVES = 2;  // one converts while the other multiplies
  struct Frag {
    bf16x8 v[4];
  };
  __device__ __forceinline__ static bf16x8 wide(int w0, int w1) {
    const bf16x2_t d[4] = {
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<uint32_t>(w0), 1.0f, false),
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<uint32_t>(w0), 1.0f, true),
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<uint32_t>(w1), 1.0f, false),
        __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<uint32_t>(w1), 1.0f, true),
    };
    return __builtin_bit_cast(bf16x8, d);
  }
  __device__ __forceinline__ static Frag frag(const i32x8& b) {
    return Frag{{wide(b[0], b[1]), wide(b[2], b[3]), wide(b[4], b[5]), wide(b[6], b[7])}};
  }
  __device__ __forceinline__ static f32x4 mac(const Frag& b, const Frag& a, f32x4 c, uint32_t sb, uint32_t sa) {
    const float z = sb == kScaleNan || sa == kScaleNan ? __uint_as_float(0x7fc00000u) : 0.0f;
    f32x4 t = {z, z, z, z};
#pragma unroll
    for (int i = 0; i < 4; ++i) t = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[i], a.v[i], t, 0, 0, 0);
    const int e = static_cast<int>(sb + sa) - 254;
#pragma unroll
    for (int r = 0; r < 4; ++r) c[r] += __builtin_amdgcn_ldexpf(t[r], e);
    return c;
  }
};

// Sums of a BM x BN tile by WM x WN waves, KS groups of them sharing the blocks
// of K: stages of KS blocks go through registers, PRE stages ahead, into a ring
// of two LDS buffers, with one barrier a stage. Both panels are rows of 128
// bytes; a stage that K cuts comes first, with zeros for the missing bytes.
// sa(i, block) is the scale byte of the lane's row in the wave's i-th tile of
// tokens, sb(h, block) that of the h-th of NB equal shares of its channels.
// Group ks has the sums of its blocks, ks, ks + KS, ...
template <class OP, int BM, int BN, int WM, int WN, int KS, int PRE, int NB, class PA, class PB, class SA, class SB>
__device__ __forceinline__ void tile_sums(int8_t (&smem)[2][(BM + BN) * KS * BK], const PA& pa, const PB& pb, int K,
                                          const SA& sa, const SB& sb, f32x4 (&acc)[BM / WM / kTile][BN / WN / kTile]) {
  constexpr int STEP = KS * BK, MI = BM / WM / kTile, NI = BN / WN / kTile, MOVES = PA::PER + PB::PER;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ks = wave / (WM * WN), wm = wave / WN % WM, wn = wave % WN;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{};
  const int cut = K % STEP, stages = (K + STEP - 1) / STEP, last_block = (K + BK - 1) / BK - 1;
  typename PA::Stage ra[PRE];
  typename PB::Stage rb[PRE];
  // stage s > 0 begins at byte (s - 1) * STEP, or s * STEP where K cuts none;
  // loads past the last stage repeat it (K >= STEP: there is a whole one)
  const int shift = cut ? STEP : 0;
  auto at = [&](int s) { return max(min(s, stages - 1) * STEP - shift, 0); };
  auto block = [&](int s) { return s == 0 && cut ? min((K - cut) / BK + ks, last_block) : at(s) / BK + ks; };
  if (PA::CUTS && cut) {
    pa.put_cut(smem[0], K - cut, K);
    pb.put_cut(smem[0] + BM * STEP, K - cut, K);
  } else {
    pa.load(ra[0], 0);
    pb.load(rb[0], 0);
    pa.put(smem[0], ra[0]);
    pb.put(smem[0] + BM * STEP, rb[0]);
  }
  auto scales = [&](int s, uint32_t (&a)[MI], uint32_t (&b)[NB]) __attribute__((always_inline)) {
    const int at_block = block(s);
#pragma unroll
    for (int i = 0; i < MI; ++i) a[i] = sa(i, at_block);
#pragma unroll
    for (int h = 0; h < NB; ++h) b[h] = sb(h, at_block);
  };
  // before the loads of stages: a loop's first wait counts what is outstanding in
  // front of it too, and scales behind them would wait for all of those
  uint32_t as[2][MI], bs[2][NB];
  scales(0, as[0], bs[0]);
#pragma unroll
  for (int u = 0; u < PRE; ++u) {
    pa.load(ra[u], at(u + 1));
    pb.load(rb[u], at(u + 1));
  }
  // vectors first .. first + count - 1 of the stage in registers R to `buf`, and
  // the stage at byte `ahead` into the registers
  auto moves = [&](auto reg, int8_t* buf, int ahead, int first, int count) __attribute__((always_inline)) {
    constexpr int R = decltype(reg)::value;
#pragma unroll
    for (int v = first; v < first + count; ++v) {
      if (v < PA::PER) {
        pa.put_one(buf, ra[R], v);
        pa.load_one(ra[R], v, ahead);
      } else if (v < MOVES) {
        pb.put_one(buf + BM * STEP, rb[R], v - PA::PER);
        pb.load_one(rb[R], v - PA::PER, ahead);
      }
    }
  };
  // a lane's bytes of a row: 16 from 16 q on, and 64 behind them
  auto bytes = [&](const int8_t* panel, int row) __attribute__((always_inline)) {
    return join32(*reinterpret_cast<const i32x4*>(panel + slot_of(row, lane >> 4)),
                  *reinterpret_cast<const i32x4*>(panel + slot_of(row, 4 + (lane >> 4))));
  };
  auto bytes_a = [&](const int8_t* buf, int i) __attribute__((always_inline)) {
    return bytes(buf + ks * BM * BK, wm * (BM / WM) + i * kTile + token_of(lane));
  };
  auto bytes_b = [&](const int8_t* buf, int j) __attribute__((always_inline)) {
    return bytes(buf + BM * STEP + ks * BN * BK, wn * (BN / WN) + j * kTile + token_of(lane));
  };
  // A stage goes tile of channels by tile of channels. Meanwhile the next one's
  // fragment is read, and stage s + 1 goes, a share at a time, from its registers
  // to LDS, where it is followed by stage s + 1 + PRE. (Reads stand before
  // writes: the compiler keeps their order.) The barrier stands behind the
  // stage's last read and before the first of the next: from there on `nxt` is
  // whole and `cur` free, and the last tile of channels hands its token fragments
  // over one by one. (All fragments of a stage read ahead in one go take the
  // registers of a second workgroup: 128 x 128 tiles, 4096^3, 113 us so, 136.)
  static_assert(NI > 1, "moves stand between tiles of channels");
  static_assert(PRE == 1 || PRE == 2, "a turn of the loop is PRE stages");
  constexpr int SHARE = (MOVES + NI - 2) / (NI - 1);  // moves a step
  typename OP::Frag fa[MI], fb;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MI; ++i) fa[i] = OP::frag(bytes_a(smem[0], i));
  fb = OP::frag(bytes_b(smem[0], 0));
  auto stage = [&](int s, auto reg) __attribute__((always_inline)) {
    const int8_t* cur = smem[s & 1];
    int8_t* nxt = smem[(s + 1) & 1];
    const int ahead = at(s + 1 + PRE);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const bool tail = j == NI - 1;
      if (tail) __syncthreads();
      const i32x8 next = tail ? bytes_b(nxt, 0) : bytes_b(cur, j + 1);
      if (j == 0) scales(s + 1, as[1], bs[1]);
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        acc[i][j] = OP::mac(fb, fa[i], acc[i][j], bs[0][j * NB / NI], as[0][i]);
        if (tail) fa[i] = OP::frag(bytes_a(nxt, i));
      }
      if (!tail) moves(reg, nxt, ahead, j * SHARE, SHARE);
      // reads first, the rest between the matrix instructions, and no step's into another's
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);  // LDS read
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // MFMA
        if (tail) {
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        } else if (i % (MI / (SHARE < MI ? SHARE : MI)) == 0) {
          __builtin_amdgcn_sched_group_barrier(0x200, (SHARE + MI - 1) / MI, 0);  // LDS write
          __builtin_amdgcn_sched_group_barrier(0x020, (SHARE + MI - 1) / MI, 0);  // global load
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      fb = OP::frag(next);
    }
#pragma unroll
    for (int i = 0; i < MI; ++i) as[0][i] = as[1][i];
#pragma unroll
    for (int h = 0; h < NB; ++h) bs[0][h] = bs[1][h];
  };
  for (int s = 0; s < stages; s += PRE) {
    stage(s, std::integral_constant<int, 0>{});
    if constexpr (PRE > 1) {
      if (s + 1 < stages) stage(s + 1, std::integral_constant<int, 1>{});
    }
  }
}

}  // namespace
