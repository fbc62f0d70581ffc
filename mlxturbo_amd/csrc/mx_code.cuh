// The MFMA tile of 4-bit by 4-bit products (qqmm): BM rows of x codes times 256
// weight rows, both as codes and scale bytes.
//
// 256 threads = 4 waves, one per SIMD, two by two: a wave owns BM / 2 rows and 128
// weight rows as 16x16 blocks.  A round is 512 codes (256 bytes) of K, four
// substeps of one 16x16x128 MFMA per block; 16 bytes of an operand are a group
// (lane (r, c): row r, group 4 q + c of the round), straight into the MFMA.
//
//  * Both operands pass LDS, by the buffer loads' LDS form in whole lines: eight
//    lanes per row and 128 bytes.  Loaded into registers in the operand's own order
//    (neighbouring lanes on different rows) each lane's 16 bytes were an access of
//    the L1 of their own, four times as many, and bound the loop: a round of 192
//    rows took 8900 cycles, 2.9 times its MFMAs' own.
//  * A stage holds two substeps (half a round; chunk p of row r stored at
//    p ^ (r & 7), so the rows of a fragment read lie in distinct banks); fragments
//    are read a substep ahead into registers, so that a half is free for the next
//    round's at the start of its second substep, behind the one barrier that says
//    the other half has landed.  A round's scale bytes travel likewise.
//  * What is not an MFMA is placed between them (sched_barrier).
//
// 4096 rows, N=17408 K=5120: 234 us in a row of calls, 3.1 PFLOP/s.  A launch by
// itself, at 2.0 GHz, 215: a round takes 2.3 us against 1.5 of MFMAs (without the loads
// of the loop 177 us, without the fragment reads 200), a tile's start and stores about
// 12.
//
// Groups past K: zero codes of x (the quantizer's padding), scale bytes 0.
#pragma once
#include "mx_common.cuh"
#include "mx_launch.h"

namespace mq {

// x rows of codes as mx_pack_kernel writes them: row m at m * steps * 256 bytes,
// padded with zero codes to whole rounds; the scales of row m and round s are 16
// bytes at (m * steps + s) * 16, byte 4 c + q that of group 16 s + 4 q + c.

template <int BM> struct MxCodeShape {
  static constexpr int kX = BM * 128;                       // bytes of x in a half
  static constexpr int kHalf = kX + 256 * 128;
  static constexpr int kScales = 256 * 16 + 256 * 16;       // x's (BM rows used), weights'
};

// xr, xs: the tile's x rows of codes and of scale bytes; w, scales: ncols weight
// rows; rounds kt0 .. kt0 + nk of the K axis.  TAIL: K is not whole rounds (rows of
// scale bytes are not 16-byte aligned).  put(i, j, v): v[e] = the sum of tile row
// BM / 2 * (wave & 1) + 16 i + r and weight row 128 * (wave >> 1) + 16 j + 4 c + e.
template <int BM, bool TAIL, class Put>
__device__ __forceinline__ void mx_code_tile(__amdgpu_buffer_rsrc_t xr, __amdgpu_buffer_rsrc_t xs,
                                             const uint32_t* __restrict__ w,
                                             const uint8_t* __restrict__ scales, int ncols, int G,
                                             int steps, int kt0, int nk, Put put,
                                             unsigned char* __restrict__ H0,
                                             unsigned char* __restrict__ H1,
                                             unsigned char* __restrict__ SC) {
  using Sh = MxCodeShape<BM>;
  constexpr int MB = BM / 32, NB = 8;           // a wave's blocks
  constexpr int XL = BM / 32, WL = 8;           // loads of a half per wave, 8 rows each
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  uint32_t skew;
  const auto rw = wide_rsrc(w, (int64_t)ncols * G * 16);
  const auto rs = mx_scale_rsrc(scales, (int64_t)ncols * G, skew);
  const uint32_t wrow = (uint32_t)G * 16u, xrow = (uint32_t)steps * 256u;
  const uint32_t chunk = 16u * (uint32_t)((lane & 7) ^ (lane >> 3));
  uint32_t wo[WL], xo[XL];
#pragma unroll
  for (int v = 0; v < WL; ++v) wo[v] = (uint32_t)(64 * wave + 8 * v + (lane >> 3)) * wrow + chunk;
#pragma unroll
  for (int v = 0; v < XL; ++v)
    xo[v] = (uint32_t)(BM / 4 * wave + 8 * v + (lane >> 3)) * xrow + chunk;
  const uint32_t xso = (uint32_t)t * (uint32_t)steps * 16u;
  const uint32_t so = t < ncols ? skew + (uint32_t)(t * G) : 0x80000000u;
  // fragment addresses of the two substeps of a half
  uint32_t fx[2], fw[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t f = r * 128 + (((4 * q + c) ^ (r & 7)) << 4);
    fx[q] = f + wm * (BM / 2) * 128;
    fw[q] = f + Sh::kX + wn * 128 * 128;
  }
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  auto half = [&](auto hc) -> unsigned char* { return decltype(hc)::value ? H1 : H0; };
  // past the last round: past every range (zeros, no traffic)
  auto at = [&](int s, uint32_t b) { return s < nk ? (uint32_t)(kt0 + s) * b : 0x80000000u; };

  // load v of half h of round s
  auto load = [&](int s, auto hc, auto vc) {
    constexpr int h = decltype(hc)::value, v = decltype(vc)::value;
    const uint32_t k = at(s, 256u) + 128u * h;
    if constexpr (v < WL)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rw, (lds_void*)(half(hc) + Sh::kX + (8 * wave + v) * 1024), 16, wo[v], k, 0, 0);
    else
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (lds_void*)(half(hc) + (XL * wave + v - WL) * 1024), 16, xo[v - WL], k, 0, 0);
  };
  // the scale bytes of round s: thread t those of x row t and of weight row t
  u32x4 sa;
  uint32_t sb;
  uint32_t sround = 0;
  auto scale_load = [&](int s) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xs, (lds_void*)(SC + wave * 1024), 16, xso,
                                             at(s, 16u), 0, 0);
    if constexpr (TAIL) {
      const uint32_t o = so == 0x80000000u || s >= nk ? 0x80000000u : so + 16u * (kt0 + s);
      sa = __builtin_amdgcn_raw_buffer_load_b128(rs, o & ~3u, 0, 0);
      sb = __builtin_amdgcn_raw_buffer_load_b32(rs, (o & ~3u) + 16u, 0, 0);
      sround = kt0 + s;
    } else {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void*)(SC + 4096 + wave * 1024), 16, so,
                                               at(s, 16u), 0, 0);
    }
  };
  // TAIL: the loaded dwords to the row's 16 bytes, those past K zero
  auto scale_store = [&]() {
    if constexpr (TAIL) {
      const uint32_t sh = so & 3u;
      u32x4 v;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        v[q] = __builtin_amdgcn_alignbyte(q < 3 ? sa[q + 1] : sb, sa[q], sh);
        const int left = G - (int)(16 * sround) - 4 * q;     // bytes that are the row's
        if (left < 4) v[q] = left > 0 ? v[q] & ((1u << (8 * left)) - 1u) : 0u;
      }
      *reinterpret_cast<u32x4*>(SC + 4096 + t * 16) = v;
    }
  };

  f32x4 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      // zeros of their own (from one shared zero the compiler copies every sum)
      asm volatile("" : "+a"(acc[i][j]));
    }
  u32x4 X[2][MB], W[2][NB], S[NB];
  uint32_t xe[MB], xn[MB], we[2][NB];
  // item v of the fragments of substep q, into register set q & 1
  auto frag = [&](auto qc, auto vc) {
    constexpr int q = decltype(qc)::value, v = decltype(vc)::value;
    using H = std::integral_constant<int, (q >> 1)>;
    if constexpr (v == 0)
      W[q & 1][0] = *reinterpret_cast<const u32x4*>(half(H{}) + fw[q & 1]);
    else if constexpr (v <= MB)
      X[q & 1][v - 1] = *reinterpret_cast<const u32x4*>(half(H{}) + fx[q & 1] + 2048 * (v - 1));
    else
      W[q & 1][v - MB] = *reinterpret_cast<const u32x4*>(half(H{}) + fw[q & 1] + 2048 * (v - MB));
  };
  auto scale_read = [&](auto vc) {
    constexpr int v = decltype(vc)::value;
    if constexpr (v < NB)
      S[v] = *reinterpret_cast<const u32x4*>(SC + 4096 + (128 * wn + 16 * v + r) * 16);
    else
      xn[v - NB] = *reinterpret_cast<const uint32_t*>(
          SC + (BM / 2 * wm + 16 * (v - NB) + r) * 16 + 4 * c);
  };
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  scale_load(0);
  static_for<0, WL + XL>([&](auto vc) { load(0, I0{}, vc); });
  static_for<0, WL + XL>([&](auto vc) { load(0, I1{}, vc); });
  scale_store();
  barrier();
  static_for<0, NB + MB>([&](auto vc) { scale_read(vc); });
  static_for<0, NB + MB>([&](auto vc) { frag(I0{}, vc); });
#pragma unroll
  for (int j = 0; j < NB; ++j) we[0][j] = S[j][0] >> (8 * c);
#pragma unroll
  for (int i = 0; i < MB; ++i) xe[i] = xn[i];

  auto substep = [&](int s, auto qc) {
    constexpr int q = decltype(qc)::value;
    using Q1 = std::integral_constant<int, (q + 1) & 3>;
    if constexpr (q & 1) barrier();
    static_for<0, NB>([&](auto jc) {
      constexpr int j = decltype(jc)::value;
      // the next substep's fragments (q = 3: the next round's)
      static_for<j * (NB + MB) / NB, (j + 1) * (NB + MB) / NB>([&](auto vc) { frag(Q1{}, vc); });
      if constexpr (q == 3)
        static_for<j * (NB + MB) / NB, (j + 1) * (NB + MB) / NB>([&](auto vc) { scale_read(vc); });
#pragma unroll
      for (int i = 0; i < MB; ++i) {
        const i32x8 a = __builtin_shufflevector(bitcast<i32x4>(W[q & 1][j]),
                                                bitcast<i32x4>(W[q & 1][j]), 0, 1, 2, 3, -1, -1,
                                                -1, -1);
        const i32x8 b = __builtin_shufflevector(bitcast<i32x4>(X[q & 1][i]),
                                                bitcast<i32x4>(X[q & 1][i]), 0, 1, 2, 3, -1, -1,
                                                -1, -1);
        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            a, b, acc[i][j], 4, 4, 0, (int)we[q & 1][j], q, (int)xe[i]);
      }
      if constexpr (q < 3) we[(q + 1) & 1][j] = S[j][q + 1] >> (8 * c);
      // the half behind the barrier is read: the next round's
      if constexpr (q & 1) {
        if constexpr (q == 1 && j == 0) scale_load(s + 1);
        static_for<j * (WL + XL) / NB, (j + 1) * (WL + XL) / NB>([&](auto vc) {
          load(s + 1, std::integral_constant<int, q / 2>{}, vc);
        });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    if constexpr (q == 2) scale_store();
    if constexpr (q == 3) {
#pragma unroll
      for (int j = 0; j < NB; ++j) we[0][j] = S[j][0] >> (8 * c);
#pragma unroll
      for (int i = 0; i < MB; ++i) xe[i] = xn[i];
    }
  };
  for (int s = 0; s < nk; ++s) {
    substep(s, I0{});
    substep(s, I1{});
    substep(s, I2{});
    substep(s, I3{});
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) put(i, j, acc[i][j]);
}

}  // namespace mq
