// Products past quantized weights: out[M, K] = d[M, N] . deq(W[N, K]), the
// gradient of x of d = x . W^T; with a second matrix the sum of two such products
// (the gated block's gate and up projections, d's halves side by side).
//
// Here the codes run along the output, and an MFMA operand wants eight weights
// along the sum.  A wave dequantizes 16 rows x its 64 columns at a time: a lane
// takes the same eight columns of two rows, rounds the two rows' weights of a column
// into one dword (so the rounding makes half of the transposition), and the dwords
// go through 2 KB of LDS of the wave's own, from which a lane reads eight weights of a
// column at once: no barrier, and a quarter of the LDS traffic of d's fragments.
// (The transposing LDS reads, ds_read_b64_tr_b16, would take the other half too, but
// the compiler has them wait for every load into LDS that is under way.)
//
// Many rows: MFMAs, at a clock that power holds near 1.8 GHz.  Both matrices of 17408 x 5120,
// 4 bits, 2048 rows of pairs 1400 - 1430 us, 1.04 PFLOP/s of MFMAs, whose pipes are busy for 63%
// of the tiles' time, and 17 for the sum of 2 splits.  One matrix of 5120 x 17408, 1024 rows
// 232 - 268 us (51%, 408 tiles on 256 CUs).  Fewer rows: the latency of a step's chain at
// one wave per SIMD (30 - 36%): 301 rows of pairs of 2 x (8192 x 2048) on 6 splits 65 + 4, 77 rows
// of 65536 x 2048 at 8 bits on 28 62 + 8.
#pragma once
#include "dense.cuh"
#include "glu_launch.h"

namespace mq {

// Dequantizing 8 columns of two rows (words wa, wb, of 8 bits two each; scales sa, sb
// times the codes' place, biases ba, bb) in pieces 0..15 of about two VALU
// instructions, run in order between MFMAs; put(k, v): v = the two rows' weights of
// column k.
template <int DT, int BITS>
struct PairPieces {
  uint32_t a, b;
  float fa, fb, ga, gb;
  template <int X, class PutPair>
  __device__ __forceinline__ void piece(uint32_t wa, uint32_t wb, float sa, float ba, float sb,
                                        float bb, PutPair&& put) {
    constexpr int q = X / 4, P = X % 4;
    if constexpr (P == 0) {
      constexpr uint32_t mask = BITS == 8 ? 0x00FF00FFu : q & 1 ? 0x00F000F0u : 0x000F000Fu;
      constexpr int shift = BITS == 8 ? (q & 1 ? 8 : 0) : (q & 2 ? 8 : 0);
      a = (wa >> shift) & mask;
      b = (wb >> shift) & mask;
    } else if constexpr (P == 1) {
      fa = __builtin_fmaf(half_lo(a), sa, ba);
      fb = __builtin_fmaf(half_lo(b), sb, bb);
    } else if constexpr (P == 2) {
      ga = __builtin_fmaf(half_hi(a), sa, ba);
      gb = __builtin_fmaf(half_hi(b), sb, bb);
    } else {
      constexpr int k = BITS == 4 ? q : 4 * (q / 2) + (q & 1);
      put(std::integral_constant<int, k>{}, T16<DT>::pack2(fa, fb));
      put(std::integral_constant<int, BITS == 4 ? k + 4 : k + 2>{}, T16<DT>::pack2(ga, gb));
    }
  }
};

// LDS of one wave behind each of the stages A0 and A2: a block of weights, and two
// steps' scales and biases (a dword per row and group).  The compiler lets a read of
// LDS wait for the loads into LDS of the same array, or, where no load goes to
// that array, for all of them.  So the reads of body steps 3 and 0 are from A0's
// part, which was last filled in step 1, and those of steps 1 and 2 from A2's.
constexpr int kGradBlock = 2048, kGradScales = 512;
constexpr int kGradWaveLds = kGradBlock + 2 * kGradScales;
// the part that body step u reads: 0 (A0) or 1 (A2)
constexpr int grad_part(int u) { return (u & 3) == 0 || (u & 3) == 3 ? 0 : 1; }

// Scalar offset of a step's rows from `row` on in a matrix of `bytes` bytes and rows of
// rowB.  A raw buffer load is in range where its lane's offset is below the buffer's size
// less the scalar offset, so that one stays within the size: a block of the last step may
// begin past the last row, and then reads zeros.
__host__ __device__ inline uint32_t grad_rows_at(uint32_t row, uint32_t rowB, int64_t bytes) {
  const uint32_t o = row * rowB;
  return o < (uint32_t)bytes ? o : (uint32_t)bytes;
}
// The first of the two rows of a block (weight rows 8 s .. + 7 and 32 + 8 s .. + 7 of a step)
// that a lane dequantizes, less 8 s.
__host__ __device__ inline uint32_t grad_lane_row(int lane) {
  return (uint32_t)(((lane & 7) >> 2) * 32 + 2 * (lane & 3));
}

// One tile: BM rows of d times 256 columns of the weights (64 per wave, as two
// 32-column blocks) over steps kt0 .. kt0 + nk - 1 (nk >= 1) of 64 weight rows, nst
// of them in each matrix.  As stream_tile.cuh's tile, d goes to LDS three steps
// ahead in four stages; the codes of a substep's 16 rows go to registers eight
// substeps ahead, a step's scales three steps ahead (and to LDS, where all lanes find
// them, a step ahead), and are dequantized two substeps before their MFMAs.
// Rows of W past N and columns past K read zeros (past the buffers' ranges).
// col0: the tile's first column; xrow_off, put and put_block as there (a tile row's
// weight rows are columns here).  PAIR: a row's sums are those of tile rows r and r + BM / 2,
// which put adds; put_block is given their sum (i < BM / 64).
template <int DT, int BITS, int GS, int BM, bool PAIR, class XRowOff, class Put, class PutBlock>
__device__ __forceinline__ void grad_tile(
    __amdgpu_buffer_rsrc_t xr, XRowOff xrow_off, const uint32_t* __restrict__ w1,
    const uint16_t* __restrict__ s1, const uint16_t* __restrict__ b1,
    const uint32_t* __restrict__ w2, const uint16_t* __restrict__ s2,
    const uint16_t* __restrict__ b2, int N, int K, int col0, int nst, int kt0, int nk, Put put,
    PutBlock put_block, unsigned char* __restrict__ A0, unsigned char* __restrict__ A1,
    unsigned char* __restrict__ A2, unsigned char* __restrict__ A3) {
  constexpr int MB = BM / 32, DM = BM / 32, NS = 2 * MB;
  constexpr int WW = BITS / 4;                  // dwords of 8 codes
  constexpr int RB = 8;                         // blocks of codes in flight
  constexpr int NG = GS == 32 ? 2 : 1;          // groups of the wave's 64 columns
  using T = T16<DT>;
  const int t = threadIdx.x, lane = t & 63;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int h = lane >> 5, lr = lane & 31;
  const int G = K / GS;
  const uint32_t rowB = (uint32_t)K * BITS / 8, rowS = (uint32_t)G * 2u;
  const int64_t wbytes = (int64_t)N * rowB, sbytes = (int64_t)N * rowS;
  // block s of a step: weight rows 8 s .. + 7 and 32 + 8 s .. + 7; this lane's are rows
  // 2 np and 2 np + 1 of the 16, its columns 8 ko .. + 7 of the wave's 64
  const int np = lane & 7, ko = lane >> 3, wc = col0 + 64 * wave;
  const uint32_t lrow = grad_lane_row(lane);
  const uint32_t wo = wc + 8 * ko < K ? lrow * rowB + (uint32_t)(wc + 8 * ko) * BITS / 8 : 0x80000000u;
  const uint32_t wo1 = wc + 8 * ko < K ? wo + rowB : 0x80000000u;
  // scales: lane l loads row l of the step
  uint32_t so[NG];
#pragma unroll
  for (int i = 0; i < NG; ++i)
    so[i] = wc + 32 * i < K ? (uint32_t)lane * rowS + (uint32_t)(wc / GS + i) * 2u : 0x80000000u;
  // Weights of column 8 ko + i lie at 256 i + 32 (ko ^ i), the 16 rows in order: a
  // store of one i writes 256 contiguous bytes, and eight columns' reads hit distinct
  // banks.
  // (offsets summed before they meet an array: the compiler follows an address to its
  // array over a few additions only)
  const uint32_t part = StreamLds<BM>::kStage + wave * kGradWaveLds;
  unsigned char *bw[2][8], *sw[2];
  const unsigned char* br[2][2];
  const unsigned char* sr[2];                   // + 32 s
  uint32_t zero;                                // see ap
  asm volatile("s_mov_b32 %0, 0" : "=s"(zero));
#pragma unroll
  for (int p = 0; p < 2; ++p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t o = zero + part + 256 * i + 32 * (ko ^ i) + 4 * np;
      bw[p][i] = (p ? A2 : A0) + o;
    }
    const uint32_t os = zero + part + kGradBlock + 4 * lane;
    sw[p] = (p ? A2 : A0) + os;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t o = zero + part + 256 * (lr & 7) + 32 * ((4 * j + (lr >> 3)) ^ (lr & 7)) + 16 * h;
      br[p][j] = (p ? A2 : A0) + o;
    }
    const uint32_t o = zero + part + kGradBlock + (NG == 2 ? 256 * (ko >> 2) : 0) + 4 * lrow;
    sr[p] = (p ? A2 : A0) + o;
  }
  uint32_t dmo[DM];
#pragma unroll
  for (int i = 0; i < DM; ++i) {
    const int r = 8 * (wave * DM + i) + (lane >> 3);
    dmo[i] = xrow_off(r) + 16u * (uint32_t)((lane & 7) ^ row_swz(r));
  }
  // (the opaque zero keeps a stage's base in the address register)
  const unsigned char* ap[4][4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const uint32_t o = lr * 128 + (((4 * h + s) ^ row_swz(lr)) << 4);
    ap[0][s] = A0 + zero + o;
    ap[1][s] = A1 + zero + o;
    ap[2][s] = A2 + zero + o;
    ap[3][s] = A3 + zero + o;
  }
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  auto xload = [&](int kt, auto sc, auto ic) {
    constexpr int S = decltype(sc)::value & 3, i = decltype(ic)::value;
    unsigned char* base = (S == 0 ? A0 : S == 1 ? A1 : S == 2 ? A2 : A3) + wave * (DM * 1024);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(xr, (lds_void*)(base + 1024 * i), 16, dmo[i],
                                             (uint32_t)(kt0 + min(kt, nk - 1)) * 128u, 0, 0);
  };
  uint32_t Wa[RB][WW], Wb[RB][WW];
  // step kt's matrix and its first weight row there
  auto place = [&](int kt, bool& second) {
    const int k = kt0 + min(kt, nk - 1);
    second = k >= nst;
    return (uint32_t)(64 * (second ? k - nst : k));
  };
  // block s of step kt into slot c
  auto bload = [&](int kt, int s, auto cc) {
    constexpr int c = decltype(cc)::value & (RB - 1);
    bool second;
    const uint32_t o = grad_rows_at(place(kt, second) + 8 * s, rowB, wbytes);
    const auto rw = wide_rsrc(second ? w2 : w1, wbytes);
    if constexpr (WW == 1) {
      Wa[c][0] = __builtin_amdgcn_raw_buffer_load_b32(rw, wo, o, 0);
      Wb[c][0] = __builtin_amdgcn_raw_buffer_load_b32(rw, wo1, o, 0);
    } else {
      const u32x2 va = __builtin_amdgcn_raw_buffer_load_b64(rw, wo, o, 0);
      const u32x2 vb = __builtin_amdgcn_raw_buffer_load_b64(rw, wo1, o, 0);
      Wa[c][0] = va[0];
      Wa[c][1] = va[1];
      Wb[c][0] = vb[0];
      Wb[c][1] = vb[1];
    }
  };
  // scales and biases of a step: registers [step & 3], then, a step before their own,
  // LDS of that step's part, slot step & 1
  uint32_t sv[4][NG], bv[4][NG];
  auto sload = [&](int kt, auto uc) {
    constexpr int u = decltype(uc)::value & 3;
    bool second;
    const uint32_t o = grad_rows_at(place(kt, second), rowS, sbytes);
    const auto rs = wide_rsrc(second ? s2 : s1, sbytes);
    const auto rb = wide_rsrc(second ? b2 : b1, sbytes);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      sv[u][i] = __builtin_amdgcn_raw_buffer_load_b16(rs, so[i], o, 0);
      bv[u][i] = __builtin_amdgcn_raw_buffer_load_b16(rb, so[i], o, 0);
    }
  };
  bool big = false;
  auto sstore = [&](auto uc) {
    constexpr int u = decltype(uc)::value & 3;
    static_for<0, NG>([&](auto ic) {
      constexpr int i = decltype(ic)::value;
      big |= needs_plain(T::to_f32((uint16_t)sv[u][i]));
      *reinterpret_cast<uint32_t*>(sw[grad_part(u - 1)] + kGradScales * (u & 1) + 256 * i) =
          sv[u][i] | bv[u][i] << 16;
    });
  };
  // scales of block c (of the body's 16): read a substep before they are used
  u32x2 sn;
  auto sread = [&](auto cc) {
    constexpr int c = decltype(cc)::value & 15;
    sn = *reinterpret_cast<const u32x2*>(sr[grad_part((c >> 2) - 1)] + kGradScales * (c >> 2 & 1) +
                                         32 * (c & 3));
  };
  GroupScale ga, gb;
  auto group = [&] {
    ga = make_group(T::to_f32((uint16_t)sn[0]), T::to_f32((uint16_t)(sn[0] >> 16)));
    gb = make_group(T::to_f32((uint16_t)sn[1]), T::to_f32((uint16_t)(sn[1] >> 16)));
  };
  PairPieces<DT, BITS> dq;
  // piece x of dequantizing block c of the body's 16, which substep c - 1 reads
  auto bpiece = [&](auto cc, auto xc) {
    constexpr int c = decltype(cc)::value & (RB - 1), part = grad_part((decltype(cc)::value - 1) >> 2);
    constexpr int x = decltype(xc)::value, word = BITS == 4 ? 0 : x / 8;
    // 4 bits: the codes at bits 4 .. 7 of their halves (mq_common.h)
    constexpr bool high = BITS == 4 && (x / 4 & 1);
    dq.template piece<x>(Wa[c][word], Wb[c][word], high ? ga.s20 : ga.s24, ga.b,
                         high ? gb.s20 : gb.s24, gb.b, [&](auto kc, uint32_t v) {
                           *reinterpret_cast<uint32_t*>(bw[part][decltype(kc)::value]) = v;
                         });
  };
  f32x16 acc[MB][2];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  u32x4 a[2][MB], b[2][2];
  // block c's fragment of block column j
  auto bread = [&](auto pc, auto cc, auto jc) {
    constexpr int p = decltype(pc)::value, j = decltype(jc)::value;
    b[p][j] = *reinterpret_cast<const u32x4*>(br[grad_part((decltype(cc)::value - 1) >> 2)][j]);
  };
  // substep c of the body's 16: the MFMAs of fragments a[c & 1], b[c & 1]; between
  // them the next substep's fragments (S: its stage), block c + 2 dequantized, and
  // the caller's items
  auto substep = [&](auto cc, auto nst_, auto item) {
    constexpr int c = decltype(cc)::value, p = c & 1, nsub = (c + 1) & 3;
    constexpr int S = decltype(nst_)::value & 3;
    using P1 = std::integral_constant<int, p ^ 1>;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(63, 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    static_for<0, NS>([&](auto tc) {
      constexpr int i = decltype(tc)::value;
      // before the next block's weights take their place
      if constexpr (i == 0) {
        bread(P1{}, std::integral_constant<int, c + 1>{}, I0{});
        bread(P1{}, std::integral_constant<int, c + 1>{}, I1{});
      }
      if constexpr (i < MB) a[p ^ 1][i] = *reinterpret_cast<const u32x4*>(ap[S][nsub] + 4096 * i);
      acc[i / 2][i % 2] = mfma32<DT>(b[p][i % 2], a[p][i / 2], acc[i / 2][i % 2]);
      if constexpr (i == 0) group();
      if constexpr (i == 1) sread(std::integral_constant<int, c + 3>{});
      static_for<i * 16 / NS, (i + 1) * 16 / NS>([&](auto xc) {
        bpiece(std::integral_constant<int, c + 2>{}, xc);
      });
      item(tc);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto barrier = [&](auto vmc) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(waitcnt_imm(decltype(vmc)::value, 0));
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  constexpr int NL = DM + 8 + 2 * NG;           // loads of a step
  static_for<0, 3>([&](auto uc) { sload(decltype(uc)::value, uc); });
  static_for<0, RB>([&](auto cc) {
    constexpr int c = decltype(cc)::value;
    bload(c / 4, c % 4, cc);
  });
  static_for<0, DM>([&](auto vc) { xload(0, I0{}, vc); });
  static_for<0, DM>([&](auto vc) { xload(1, I1{}, vc); });
  static_for<0, DM>([&](auto vc) { xload(2, I2{}, vc); });
  // block 0 to its fragments, block 1
  sstore(I0{});
  sread(I0{});
  group();
  static_for<0, 16>([&](auto xc) { bpiece(I0{}, xc); });
  bread(I0{}, I0{}, I0{});
  bread(I0{}, I0{}, I1{});
  sread(I1{});
  group();
  static_for<0, 16>([&](auto xc) { bpiece(I1{}, xc); });
  sread(I2{});
  // stages 0 and 1: what step 0 counts on leaves out the loads before the loop
  barrier(std::integral_constant<int, DM>{});
  bload(2, 0, I0{});
  bload(2, 1, I1{});
  static_for<0, MB>([&](auto ic) {
    constexpr int i = decltype(ic)::value;
    a[0][i] = *reinterpret_cast<const u32x4*>(ap[0][0] + 4096 * i);
  });

  // step kt at place u of the body's four; nvm: the loads of one step that the wait
  // before the barrier may count on
  auto step = [&](int kt, auto uc, auto nvm) {
    constexpr int u = decltype(uc)::value;
    using N1 = std::integral_constant<int, (u + 1) & 3>;
    using N3 = std::integral_constant<int, (u + 3) & 3>;
    // substep s: its share of the loads of d of step kt + 3 (three substeps), and,
    // once they are dequantized, the codes that follow block s + 2 by eight blocks
    auto loads = [&](auto sc, auto tc) {
      constexpr int s = decltype(sc)::value, i = decltype(tc)::value, q = s * NS + i;
      if constexpr (s < 3)
        static_for<q * DM / (3 * NS), (q + 1) * DM / (3 * NS)>([&](auto vc) { xload(kt + 3, N3{}, vc); });
      if constexpr (s == 0 && i == 2) sstore(N1{});
      if constexpr (s == 1 && i == 2) sload(kt + 3, N3{});
      if constexpr (i == NS - 1)
        bload(kt + 2 + (s + 2) / 4, (s + 2) % 4, std::integral_constant<int, 4 * u + s + 2>{});
    };
    using C0 = std::integral_constant<int, 4 * u>;
    using C1 = std::integral_constant<int, 4 * u + 1>;
    using C2 = std::integral_constant<int, 4 * u + 2>;
    using C3 = std::integral_constant<int, 4 * u + 3>;
    substep(C0{}, uc, [&](auto tc) { loads(I0{}, tc); });
    substep(C1{}, uc, [&](auto tc) { loads(I1{}, tc); });
    substep(C2{}, uc, [&](auto tc) { loads(I2{}, tc); });
    barrier(std::integral_constant<int, 2 * decltype(nvm)::value>{});
    substep(C3{}, N1{}, [&](auto tc) { loads(I3{}, tc); });
  };
  // whole fours in a loop that is left at its end alone, as in stream_tile.cuh
  using Counted = std::integral_constant<int, NL>;
  using Sure = std::integral_constant<int, DM>;
  const int n4 = nk & ~3;
  int kt = 0;
  if (n4 > 0) {
    do {
      step(kt, I0{}, Counted{});
      step(kt + 1, I1{}, Counted{});
      step(kt + 2, I2{}, Counted{});
      step(kt + 3, I3{}, Counted{});
      kt += 4;
    } while (kt < n4);
  }
  if (kt < nk) {
    step(kt, I0{}, Sure{});
    if (kt + 1 < nk) {
      step(kt + 1, I1{}, Sure{});
      if (kt + 2 < nk) step(kt + 2, I2{}, Sure{});
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(waitcnt_imm(0, 0));
  asm volatile("" ::: "memory");
  if (!__syncthreads_or(big)) {
    put(acc);
    return;
  }
  // a scale of 2^100 or more: block by block, code by code from global memory
  constexpr int PB = PAIR ? MB / 2 : MB;
  for (int i = 0; i < PB; ++i) {
    for (int j = 0; j < 2; ++j) {
      f32x16 s;
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.f;
      const int col = col0 + 64 * wave + 32 * j + lr;
      for (int k = kt0; k < kt0 + nk; ++k) {
        const bool second = k >= nst;
        const auto rw = wide_rsrc(second ? w2 : w1, wbytes);
        const auto rs = wide_rsrc(second ? s2 : s1, sbytes);
        const auto rb = wide_rsrc(second ? b2 : b1, sbytes);
        for (int q = 0; q < 4; ++q) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t n = (uint32_t)(64 * (second ? k - nst : k) + 32 * h + 8 * q + e);
            const uint32_t in = col < K ? 0u : 0x80000000u;
            const uint32_t code =
                __builtin_amdgcn_raw_buffer_load_b8(rw, in | (n * rowB + (uint32_t)col * BITS / 8),
                                                    0, 0);
            const uint16_t s16 =
                __builtin_amdgcn_raw_buffer_load_b16(rs, in | (n * rowS + (uint32_t)(col / GS) * 2u),
                                                     0, 0);
            const uint16_t b16 =
                __builtin_amdgcn_raw_buffer_load_b16(rb, in | (n * rowS + (uint32_t)(col / GS) * 2u),
                                                     0, 0);
            const uint32_t c = BITS == 8 ? code : (code >> (4 * (col & 1))) & 15u;
            v[e] = __builtin_fmaf((float)c, T::to_f32(s16), T::to_f32(b16));
          }
          const u32x4 wv = {T::pack2(v[0], v[1]), T::pack2(v[2], v[3]), T::pack2(v[4], v[5]),
                            T::pack2(v[6], v[7])};
          for (int r = 32 * i + lr; r < BM; r += 32 * PB)
            s = mfma32<DT>(wv, __builtin_amdgcn_raw_buffer_load_b128(
                                   xr, xrow_off(r) + 64u * h + 16u * q, k * 128, 0), s);
        }
      }
      put_block(i, j, s);
    }
  }
}

// Grid (ceil(K / 256), ceil(M / BM), splits), 256 threads.  d: rows of ld elements, of
// which 64 nst are read.  With part, split z sums its share of the steps into the float
// plane part[z] ([M, K]) for wide_reduce_kernel; else (splits == 1) the sums are rounded
// into out.
// PAIR: both matrices, and d as two T numbers whose sum is a value (glu_grad.hip): rows of
// the first matrix's columns and the second's, 64 nst of each, then the second numbers in the
// same order.  A tile is then BM / 2 rows, the first numbers in its upper half and the second
// in its lower, whose sums are added in registers; grid.y = ceil(M / (BM / 2)).  In float16
// row m's sums are multiplied by undo[m].
template <int DT, int BITS, int GS, int BM, bool PAIR>
__global__ __launch_bounds__(256, BM <= 64 ? 2 : 1) void qmm_grad_kernel(
    const uint16_t* __restrict__ d, int64_t ld, const uint32_t* __restrict__ w1,
    const uint16_t* __restrict__ s1, const uint16_t* __restrict__ b1,
    const uint32_t* __restrict__ w2, const uint16_t* __restrict__ s2,
    const uint16_t* __restrict__ b2, const float* __restrict__ undo, uint16_t* __restrict__ out,
    float* __restrict__ part, int M, int N, int K, int nst, int splits) {
  __shared__ __align__(16) unsigned char A0[StreamLds<BM>::kStage + 4 * kGradWaveLds];
  __shared__ __align__(16) unsigned char A1[StreamLds<BM>::kStage];
  __shared__ __align__(16) unsigned char A2[StreamLds<BM>::kStage + 4 * kGradWaveLds];
  __shared__ __align__(16) unsigned char A3[StreamLds<BM>::kStage];
  constexpr int R = grad_tile_rows(BM, PAIR);
  const int m0 = blockIdx.y * R, n0 = blockIdx.x * 256;
  const int mrows = min(R, M - m0), ncols = min(256, K - n0);
  const int ns = nst * (PAIR ? 2 : 1), z = blockIdx.z;
  const int kt0 = (int)((int64_t)ns * z / splits), kt1 = (int)((int64_t)ns * (z + 1) / splits);
  const int lane = threadIdx.x & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto xr = wide_rsrc(d + (int64_t)m0 * ld,
                            ((int64_t)(mrows - 1) * ld + 64 * (PAIR ? 2 * ns : ns)) * 2);
  auto xrow_off = [&](int r) {
    const int low = PAIR && r >= R;             // the value's second number
    return (uint32_t)(min(r - (low ? R : 0), mrows - 1) * ld) * 2u + (low ? 128u * ns : 0u);
  };
  const bool vec = (uintptr_t)out % 16 == 0;    // K is whole eights
  // the sums of tile row r (the last of the tile past M)
  auto scaled = [&](int r, const f32x16& v) {
    if constexpr (PAIR && DT == kF16) return v * undo[m0 + min(r, mrows - 1)];
    else return v;
  };
  auto put_block = [&](int i, int j, const f32x16& sums) {
    const int r = 32 * i + lr;
    if (r >= mrows) return;
    const f32x16 acc = scaled(r, sums);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 64 * wave + 32 * j + 8 * q + 4 * h;
      if (c >= ncols) continue;                 // ncols is whole fours
      if (part) {
        *reinterpret_cast<f32x4*>(part + ((int64_t)z * M + m0 + r) * K + n0 + c) =
            (f32x4){acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
      } else {
        uint16_t* o = out + (int64_t)(m0 + r) * K + n0 + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = T16<DT>::round1(acc[4 * q + e]);
      }
    }
  };
  auto put = [&](f32x16 (&acc)[BM / 32][2]) {
    // read each accumulator where it is stored, not all of them before
    auto pin = [&](f32x16& v) {
      if constexpr (BM >= 128) asm volatile("" : "+a"(v));
    };
    auto sums = [&](int i, int j) {
      pin(acc[i][j]);
      if constexpr (PAIR) {
        pin(acc[i + R / 32][j]);
        return acc[i][j] + acc[i + R / 32][j];
      } else {
        return acc[i][j];
      }
    };
    if (part || !vec) {
#pragma unroll
      for (int i = 0; i < R / 32; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          put_block(i, j, sums(i, j));
          __builtin_amdgcn_sched_barrier(0);
        }
      return;
    }
    // through the wave's own stage of LDS, so that a store instruction writes
    // 128 contiguous bytes of 8 rows
    unsigned char* L = wave == 0 ? A0 : wave == 1 ? A1 : wave == 2 ? A2 : A3;
#pragma unroll
    for (int i = 0; i < R / 32; ++i) {
      const int r = 32 * i + lr;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const f32x16 v = scaled(r, sums(i, j));
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<u32x2*>(L + r * 128 + (((4 * j + q) ^ row_swz(r)) << 4) + 8 * h) =
              (u32x2){T16<DT>::pack2(v[4 * q], v[4 * q + 1]),
                      T16<DT>::pack2(v[4 * q + 2], v[4 * q + 3])};
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int c = 64 * wave + 8 * (lane & 7);
    uint16_t* ot = out + (int64_t)m0 * K + n0 + c;
#pragma unroll 4
    for (int i = 0; i < R / 8; ++i) {
      const int r = 8 * i + (lane >> 3);
      const u32x4 v =
          *reinterpret_cast<const u32x4*>(L + r * 128 + (((lane & 7) ^ row_swz(r)) << 4));
      if (r < mrows && c < ncols) *reinterpret_cast<u32x4*>(ot + (int64_t)r * K) = v;
    }
  };
  grad_tile<DT, BITS, GS, BM, PAIR>(xr, xrow_off, w1, s1, b1, w2, s2, b2, N, K, n0, nst, kt0,
                                    kt1 - kt0, put, put_block, A0, A1, A2, A3);
}

template <int DT, int BITS, int GS>
int GradLaunch<DT, BITS, GS>::run(const GradArgs& a, const WidePlan& plan, void* ws,
                                  hipStream_t st, int* nlaunch) {
  float* part = plan.splits > 1 ? static_cast<float*>(ws) : nullptr;
  auto pair = [&](auto bmc, auto pairc) {
    constexpr int BM = decltype(bmc)::value, R = grad_tile_rows(BM, decltype(pairc)::value);
    const dim3 grid((unsigned)((a.K + 255) / 256), (unsigned)((a.M + R - 1) / R),
                    (unsigned)plan.splits);
    hipLaunchKernelGGL((qmm_grad_kernel<DT, BITS, GS, BM, decltype(pairc)::value>), grid,
                       dim3(256), 0, st, (const uint16_t*)a.d, a.ld, a.w1, (const uint16_t*)a.s1,
                       (const uint16_t*)a.b1, a.w2, (const uint16_t*)a.s2, (const uint16_t*)a.b2,
                       a.undo, (uint16_t*)a.out, part, (int)a.M, (int)a.N, (int)a.K,
                       (int)grad_steps(a.N), plan.splits);
  };
  auto go = [&](auto bmc) {
    if (a.w2) pair(bmc, std::true_type{});
    else pair(bmc, std::false_type{});
  };
  switch (plan.bm) {
    case 64: go(std::integral_constant<int, 64>{}); break;
    case 128: go(std::integral_constant<int, 128>{}); break;
    case 192: go(std::integral_constant<int, 192>{}); break;
    default: go(std::integral_constant<int, 256>{}); break;
  }
  *nlaunch += 1;
  if (part) {
    const int64_t MK = a.M * a.K;
    const auto kern = (uintptr_t)a.out % 8 == 0 ? wide_reduce_kernel<DT, true>
                                                : wide_reduce_kernel<DT, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)((MK + 1023) / 1024)), dim3(256), 0, st, part,
                       (uint16_t*)a.out, MK, plan.splits);
    *nlaunch += 1;
  }
  return 0;
}

}  // namespace mq
