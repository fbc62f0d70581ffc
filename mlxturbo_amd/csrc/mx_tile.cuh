// The MFMA tile of wide MXFP4 products with x of 16 bits: BM rows of x times 256
// weight rows.
//
// 256 threads = 4 waves, one per SIMD (two workgroups per CU at BM = 64); a
// wave owns all BM rows and 64 weight rows as four 16-row blocks.  A step is 128
// values of K (256 bytes of an x row), four substeps q; per substep and 16-row
// block of x ("slot") a wave runs four 16x16x32 MFMAs, one per weight block, of 16
// cycles each.
//
//  * Lane (r = lane & 15, c = lane >> 4) of an operand holds row r: 16 bytes of
//    weights are its group c of the step's four, word q the 8 codes of substep q,
//    converted by four instructions of two codes into the MFMA's operand; the x
//    chunk is 4 c + q.
//  * x goes to LDS by the buffer loads' LDS form, ST - 1 steps ahead in ST
//    stages (whole 256-byte row pieces; chunk p of row r stored at p ^ (r & 15),
//    so the 16 rows of a fragment read lie in distinct banks); weights and their
//    scale bytes to registers, as far ahead.  Weights never pass LDS: each is
//    read and converted once per tile.
//  * Fragments are read kAhead slots before their MFMAs.  The reads of the next
//    step's first slots lie behind one barrier per step, at slot SLOTS - kAhead,
//    where the next step's x has landed and every wave has read the last of
//    this step's, so the stage may be refilled.
//  * What is not an MFMA (fragment reads, conversions, loads) is placed between
//    them slot by slot (sched_barrier): a wave runs alone on its SIMD.
//
// Groups past K: zero codes and scale bytes 0, x zero (outside the buffer ranges).
#pragma once
#include "mx_common.cuh"
#include "mx_launch.h"

namespace mq {

template <int BM> struct MxTileShape {
  static constexpr int kStages = BM >= 192 ? 2 : 4;
  static constexpr int kStage = BM * 256;                // bytes of x
};

// xoff(r): byte offset of tile row r in xr, or 0x80000000 (zeros).  TAIL: K is not
// whole 512s (rows of scale bytes are not 16-byte aligned, and steps may end in the
// middle).  Without TAIL: kt0 and nk in whole rounds of kStages steps.
// put(i, j, v): v[e] = the sum of tile row 16 i + r and the wave's weight row 16
// j + 4 c + e.
template <int DT, int BM, bool TAIL, class XOff, class Put>
__device__ __forceinline__ void mx_tile(__amdgpu_buffer_rsrc_t xr, XOff xoff,
                                        const uint32_t* __restrict__ w,
                                        const uint8_t* __restrict__ scales, int ncols, int G,
                                        int kt0, int nk, Put put, unsigned char* __restrict__ A0,
                                        unsigned char* __restrict__ A1,
                                        unsigned char* __restrict__ A2,
                                        unsigned char* __restrict__ A3) {
  constexpr int ST = MxTileShape<BM>::kStages, MB = BM / 16, SLOTS = 4 * MB, DM = BM / 16;
  // slots a fragment is read ahead, and fragment registers
  constexpr int P = MB == 1 ? 2 : MB <= 4 ? 3 : 6, R = MB == 1 ? 4 : 8;
  static_assert(SLOTS % R == 0 && P < R, "a step's slots run through whole rings");
  constexpr int SQ = TAIL ? 1 : 0;              // scale loads per block and step
  constexpr int NW = 4 + 4 * SQ, NL = NW + DM;  // loads of weights, of all, per wave and step
  // Steps of weights and of their scale bytes in registers, as many as the sums
  // leave room for (64 rows: with two, a step waited for the weights of the
  // step before it).
  constexpr int WR = BM >= 192 ? 2 : 4;
  constexpr bool PAIR = WR == 4;
  using T = T16<DT>;
  const int t = threadIdx.x, lane = t & 63, r = lane & 15, c = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  uint32_t skew;
  const auto rw = wide_rsrc(w, (int64_t)ncols * G * 16);
  const auto rs = mx_scale_rsrc(scales, (int64_t)ncols * G, skew);
  uint32_t wo[4], so[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = 64 * wave + 16 * j + r;
    wo[j] = (uint32_t)(row * G + c) * 16u;
    so[j] = row < ncols ? skew + (uint32_t)(row * G + (TAIL ? c : 0)) : 0x80000000u;
  }
  // fragment addresses per stage and substep; the opaque zero keeps a stage's
  // base in the address register, since an offset field reaches 64 KB only
  uint32_t zero;
  asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
  auto stage = [&](auto sc) -> unsigned char* {
    constexpr int S = decltype(sc)::value % ST;
    return S == 0 ? A0 : S == 1 ? A1 : S == 2 ? A2 : A3;
  };
  uint32_t fo[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) fo[q] = zero + r * 256 + (((4 * c + q) ^ r) << 4);
  uint32_t dmo[DM];

  u32x4 W[WR][4];
  uint32_t S[WR][4];                            // TAIL: scale bytes
  // Whole rounds: a round's scale bytes (four per step) in one load per block.
  // Byte loads for every step brought each row's line to the L1 again, as much
  // as the weights (N=5120 K=17408, 45 rows, 12 splits: 40 against 32 us).
  uint32_t cur[4][ST], nxt[4][ST];
  auto sround = [&](int s, uint32_t (&d)[4][ST]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t o = s < nk ? (uint32_t)(kt0 + s) * 4u : 0x80000000u;
      if constexpr (ST == 4) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(rs, so[j], o, 0);
#pragma unroll
        for (int i = 0; i < ST; ++i) d[j][i] = v[i];
      } else {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(rs, so[j], o, 0);
#pragma unroll
        for (int i = 0; i < ST; ++i) d[j][i] = v[i];
      }
    }
  };
  // byte offset of step s in rows of b bytes a step; past the last step, past
  // every range (zeros, no traffic)
  auto at = [&](int s, uint32_t b) { return s < nk ? (uint32_t)(kt0 + s) * b : 0x80000000u; };
  // item v of the loads of step s, into stage / ring slot sc
  auto load = [&](int s, auto sc, auto vc) {
    constexpr int v = decltype(vc)::value, SW = decltype(sc)::value % WR;
    const int k = kt0 + s;
    if constexpr (v < 4) {
      uint32_t o = wo[v];
      if constexpr (TAIL) o = 4 * k + c < G ? o : 0x80000000u;
      W[SW][v] = __builtin_amdgcn_raw_buffer_load_b128(rw, o, at(s, 64u), 0);
    } else if constexpr (v < NW) {
      const uint32_t o = 4 * k + c < G ? so[v - 4] : 0x80000000u;
      S[SW][v - 4] = __builtin_amdgcn_raw_buffer_load_b8(rs, o, at(s, 4u), 0);
    } else {
      constexpr int i = v - NW;
      uint32_t o = dmo[i];
      if constexpr (TAIL) {
        const int p = (lane & 15) ^ (4 * ((wave * DM + i) & 3) + (lane >> 4));
        o = 4 * k + (p >> 2) < G ? o : 0x80000000u;
      }
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (lds_void*)(stage(sc) + (wave * DM + i) * 1024), 16, o, at(s, 256u), 0, 0);
    }
  };

  f32x4 acc[MB][4];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
      // zeros of their own: from one shared zero the compiler made the first
      // MFMA of every sum in the loop read a copy (192 moves and their waits
      // per 384 MFMAs; M=2048 316 against 272 us)
      if constexpr (BM > 64) asm volatile("" : "+a"(acc[i][j]));
    }
  u32x4 A[R];
  u32x4 B[2][4];                                // weight operands of a substep
  float sf[4];
  auto frag = [&](auto sc, auto tc) {           // fragment of slot t of stage sc
    constexpr int t = decltype(tc)::value, q = t / MB, i = t % MB;
    A[t % R] = *reinterpret_cast<const u32x4*>(stage(sc) + fo[q] + 4096 * i);
  };
  // piece x of 16 of the operands of substep q from ring slot sw into B[q & 1]
  auto piece = [&](auto swc, auto qc, auto xc) {
    constexpr int u = decltype(swc)::value, q = decltype(qc)::value;
    constexpr int x = decltype(xc)::value, j = x / 4, e = x % 4;
    if constexpr (q == 0 && e == 0)
      sf[j] = mx_scale(TAIL ? S[u % WR][j] : (cur[j][u % ST] >> (8 * c)) & 255u);
    B[q & 1][j][e] = mx_pair<DT, e>(W[u % WR][j][q], sf[j]);
  };
  auto barrier = [&](auto vmc) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(decltype(vmc)::value, 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;

  // prologue: the weights first (x rows may have to be looked up)
  if constexpr (!TAIL) sround(0, cur);
  static_for<0, NW>([&](auto vc) { load(0, I0{}, vc); });
  static_for<0, NW>([&](auto vc) { load(1, I1{}, vc); });
  if constexpr (WR == 4) {
    static_for<0, NW>([&](auto vc) { load(2, I2{}, vc); });
    static_for<0, NW>([&](auto vc) { load(3, I3{}, vc); });
  }
#pragma unroll
  for (int i = 0; i < DM; ++i) {
    const int row = 4 * (wave * DM + i) + (lane >> 4);
    dmo[i] = xoff(row) + 16u * (uint32_t)((lane & 15) ^ (row & 15));
  }
  static_for<NW, NL>([&](auto vc) { load(0, I0{}, vc); });
  if constexpr (ST > 2) {
    static_for<NW, NL>([&](auto vc) { load(1, I1{}, vc); });
    static_for<NW, NL>([&](auto vc) { load(2, I2{}, vc); });
  }
  // all of it, also the x of steps 1 and 2: the first steps have fewer loads behind
  // it than Flight counts
  barrier(I0{});
  static_for<0, P>([&](auto tc) { frag(I0{}, tc); });
  static_for<0, 16>([&](auto xc) { piece(I0{}, I0{}, xc); });

  // A step issues, in this order: in its first substep the x of step s + ST - 1; in
  // the last substep, before the barrier, the weights of step s + WR, or, PAIR, in
  // every second step's those of the next two steps' successors.  Flight: those
  // issued after the x of step s + 1, which the wait before the barrier may leave in
  // flight.
  constexpr int FREE = SLOTS - P;
  constexpr int kFlight = ST == 2 ? NW : 2 * DM + 2 * NW;
  using Flight = std::integral_constant<int, (kFlight < 63 ? kFlight : 63)>;
  // one step; u: its stage
  auto step = [&](int s, auto uc) {
    constexpr int u = decltype(uc)::value;
    using U = std::integral_constant<int, u>;
    using N1 = std::integral_constant<int, u + 1>;
    using XN = std::integral_constant<int, u + ST - 1>;
    static_for<0, SLOTS>([&](auto tc) {
      constexpr int t = decltype(tc)::value, q = t / MB, i = t % MB;
      if constexpr (t == FREE) barrier(Flight{});
      if constexpr (t + P < SLOTS) frag(U{}, std::integral_constant<int, t + P>{});
      else frag(N1{}, std::integral_constant<int, t + P - SLOTS>{});
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = T::mfma(B[q & 1][j], A[t % R], acc[i][j]);
      if constexpr (!TAIL) {
        if constexpr (u == 0 && q == 1 && i == 0) sround(s + ST, nxt);
        if constexpr (u == ST - 1 && q == 3 && i == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int k = 0; k < ST; ++k) cur[j][k] = nxt[j][k];
        }
      }
      // the next substep's operands
      static_for<i * 16 / MB, (i + 1) * 16 / MB>([&](auto xc) {
        if constexpr (q < 3) piece(U{}, std::integral_constant<int, q + 1>{}, xc);
        else piece(N1{}, I0{}, xc);
      });
      if constexpr (q == 0)
        static_for<i * (NL - NW) / MB, (i + 1) * (NL - NW) / MB>([&](auto vc) {
          load(s + ST - 1, XN{}, std::integral_constant<int, NW + decltype(vc)::value>{});
        });
      if constexpr (PAIR) {
        // both halves of a line together, in the second step of a pair
        if constexpr (q == 3 && (u & 1))
          static_for<i * NW / MB, (i + 1) * NW / MB>([&](auto vc) {
            load(s + 3, std::integral_constant<int, u + 3>{}, vc);
            load(s + 4, std::integral_constant<int, u + 4>{}, vc);
          });
      } else if constexpr (q == 3 && t < FREE) {
        constexpr int n = MB - P;
        static_for<i * NW / n, (i + 1) * NW / n>([&](auto vc) {
          load(s + WR, std::integral_constant<int, u + WR>{}, vc);
        });
      }
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  // Whole rounds of the stages, in a loop that is left at its end alone (left
  // in its middle, loads into registers may be moved past the exits, and no
  // longer run ahead): steps past the last add zeros.
  for (int s = 0; s < nk; s += ST) {
    step(s, I0{});
    step(s + 1, I1{});
    if constexpr (ST == 4) {
      step(s + 2, I2{});
      step(s + 3, I3{});
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) put(i, j, acc[i][j]);
}

}  // namespace mq
