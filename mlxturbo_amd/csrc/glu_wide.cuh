// The dense gated feed-forward block of many rows: stream_tile.cuh's tile with a
// wave's two 32-row blocks on the gate and the up matrix, so that a lane holds
// both sums of its outputs and each x tile is read once for both.
//
// Many rows: MFMAs, at a clock that power holds near 1.8 GHz, as the plain product's tile
// (dense.cuh): M=2048 N=17408 K=5120 640 - 680 us, 1.07 - 1.14 PFLOP/s (a library product of that
// size 650, over weights already dequantized); the MFMA pipes are busy for 71% of the tiles'
// time, and 1088 tiles take 5 rounds of 256 CUs, the last a quarter full.  Few rows are bound
// by the latency of a tile's steps (MFMAs 19%, VALU 28%) and the sum of the splits: N=9001
// K=2560, 8 bits, 45 rows on 3 splits 19.9 + 4.0 us.
#pragma once
#include "glu.cuh"

namespace mq {

// Grid (ceil(N / 128), ceil(M / BM), splits), 256 threads; ranges as in dense.cuh.
// part: split z's sums of its share of the k-steps (whole U) go to the float planes
// part[2 z] (gate) and part[2 z + 1] (up), [M, glu_plane(N)], for glu_reduce_kernel; else
// (splits == 1) out = act(gate) * up, and the sums to gf and uf where they are given.
template <int DT, int BITS, int GS, int BM, int U>
__global__ __launch_bounds__(256, BM <= 64 ? 2 : 1) void glu_wide_kernel(
    const uint16_t* __restrict__ x, const uint32_t* __restrict__ wg,
    const uint16_t* __restrict__ sg, const uint16_t* __restrict__ bg,
    const uint32_t* __restrict__ wu, const uint16_t* __restrict__ su,
    const uint16_t* __restrict__ bu, uint16_t* __restrict__ out, float* __restrict__ gf,
    float* __restrict__ uf, float* __restrict__ part, int M, int N, int K, int act, int splits) {
  __shared__ __align__(16) unsigned char A0[StreamLds<BM>::kStage];
  __shared__ __align__(16) unsigned char A1[StreamLds<BM>::kStage];
  __shared__ __align__(16) unsigned char A2[StreamLds<BM>::kStage];
  __shared__ __align__(16) unsigned char A3[StreamLds<BM>::kStage];
  using T = T16<DT>;
  const int m0 = blockIdx.y * BM, n0 = blockIdx.x * 128;
  const int mrows = min(BM, M - m0), ncols = min(128, N - n0);
  const int64_t G = K / GS;
  const int nu = K / (64 * U), z = blockIdx.z;
  const int kt0 = U * (int)((int64_t)nu * z / splits);
  const int kt1 = U * (int)((int64_t)nu * (z + 1) / splits);
  const int lane = threadIdx.x & 63, lr = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const auto xr = wide_rsrc(x + (int64_t)m0 * K, (int64_t)mrows * K * 2);
  auto xrow_off = [&](int r) { return (uint32_t)min(r, mrows - 1) * (uint32_t)K * 2u; };
  const int64_t ld = part ? glu_plane(N) : N;   // of the sums' rows
  float* fg = part ? part + 2 * z * M * ld : gf;
  float* fu = part ? part + (2 * z + 1) * M * ld : uf;
  const bool vec = N % 8 == 0 && (uintptr_t)out % 16 == 0 && (uintptr_t)fg % 16 == 0 &&
                   (uintptr_t)fu % 16 == 0;
  // four columns of both sums (of planes: up to the padding)
  auto put_sums = [&](int64_t o, int c, const f32x4& g, const f32x4& u) {
    if (part || vec) {
      if (c < ncols) {
        *reinterpret_cast<f32x4*>(fg + o) = g;
        *reinterpret_cast<f32x4*>(fu + o) = u;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < ncols) {
          fg[o + e] = g[e];
          fu[o + e] = u[e];
        }
    }
  };
  auto quarter = [](const f32x16& a, int q) {
    return (f32x4){a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]};
  };
  auto put_rows = [&](int i, const f32x16& g, const f32x16& u, bool values) {
    const int r = 32 * i + lr;
    if (r >= mrows) return;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * wave + 8 * q + 4 * h;
      const int64_t o = (int64_t)(m0 + r) * N + n0 + c;
      const f32x4 gq = quarter(g, q), uq = quarter(u, q);
      if (fg) put_sums((m0 + r) * ld + n0 + c, c, gq, uq);
      if (values) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (c + e < ncols) out[o + e] = T::round1(glu_act(gq[e], act) * uq[e]);
      }
    }
  };
  f32x16 held;                                  // plain route: block 0 until block 1 is there
  auto put_block = [&](int i, int j, const f32x16& acc) {
    if (j == 0) held = acc;
    else put_rows(i, held, acc, !part);
  };
  auto put = [&](f32x16 (&acc)[BM / 32][2]) {
    // read each accumulator where it is stored, not all of them before
    auto pin = [&](f32x16& v) {
      if constexpr (BM >= 128) asm volatile("" : "+a"(v));
    };
    if (part || !vec) {
#pragma unroll
      for (int i = 0; i < BM / 32; ++i) {
        pin(acc[i][0]);
        pin(acc[i][1]);
        put_rows(i, acc[i][0], acc[i][1], !part);
        __builtin_amdgcn_sched_barrier(0);
      }
      return;
    }
    // through the wave's own stage of LDS, so that a store instruction writes
    // whole 64-byte pieces of rows
    unsigned char* L = wave == 0 ? A0 : wave == 1 ? A1 : wave == 2 ? A2 : A3;
#pragma unroll
    for (int i = 0; i < BM / 32; ++i) {
      const int r = 32 * i + lr;
      pin(acc[i][0]);
      pin(acc[i][1]);
      if (fg) put_rows(i, acc[i][0], acc[i][1], false);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = glu_act(acc[i][0][4 * q + e], act) * acc[i][1][4 * q + e];
        *reinterpret_cast<u32x2*>(L + r * 128 + ((q ^ row_swz(r)) << 4) + 8 * h) =
            (u32x2){T::pack2(v[0], v[1]), T::pack2(v[2], v[3])};
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int ch = lane & 3, c = 32 * wave + 8 * ch;
    uint16_t* ot = out + (int64_t)m0 * N + n0 + c;
#pragma unroll 4
    for (int i = 0; i < BM / 16; ++i) {
      const int r = 16 * i + (lane >> 2);
      const u32x4 v = *reinterpret_cast<const u32x4*>(L + r * 128 + ((ch ^ row_swz(r)) << 4));
      if (r < mrows && c < ncols) *reinterpret_cast<u32x4*>(ot + (int64_t)r * N) = v;
    }
  };
  const int64_t w0 = (int64_t)n0 * K * BITS / 32;
  stream_tile<DT, BITS, GS, BM, U, true>(xr, xrow_off, wg + w0, sg + n0 * G, bg + n0 * G, wu + w0,
                                         su + n0 * G, bu + n0 * G, ncols, K, kt0, kt1 - kt0, put,
                                         put_block, A0, A1, A2, A3);
}

// out = act(sum of the gate planes) * (sum of the up planes), in split order; four
// elements of a row per thread, quads = M * glu_plane(N) / 4 of them, 256 threads.  VEC: N in
// whole eights, out 8-byte and gf and uf 16-byte aligned.
template <int DT, bool VEC>
__global__ __launch_bounds__(256) void glu_reduce_kernel(const float* __restrict__ part,
                                                         uint16_t* __restrict__ out,
                                                         float* __restrict__ gf,
                                                         float* __restrict__ uf, uint32_t quads,
                                                         int N, int splits, int act) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= quads) return;
  const f32x4* p = reinterpret_cast<const f32x4*>(part) + i;
  const int64_t plane = quads;
  f32x4 g = p[0], u = p[plane];
  for (int z = 1; z < splits; ++z) {
    g += p[2 * z * plane];
    u += p[(2 * z + 1) * plane];
  }
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = glu_act(g[e], act) * u[e];
  if constexpr (VEC) {
    const int64_t o = 4 * (int64_t)i;
    *reinterpret_cast<u32x2*>(out + o) =
        (u32x2){T16<DT>::pack2(v[0], v[1]), T16<DT>::pack2(v[2], v[3])};
    if (gf) {
      *reinterpret_cast<f32x4*>(gf + o) = g;
      *reinterpret_cast<f32x4*>(uf + o) = u;
    }
  } else {
    const uint32_t per = (uint32_t)glu_plane(N) / 4, r = i / per;
    const int c = 4 * (int)(i - r * per);
    const int64_t o = (int64_t)r * N + c;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (c + e < N) {
        out[o + e] = T16<DT>::round1(v[e]);
        if (gf) {
          gf[o + e] = g[e];
          uf[o + e] = u[e];
        }
      }
    }
  }
}

template <int DT, int BITS, int GS>
int GluWideLaunch<DT, BITS, GS>::run(const GluArgs& a, const WidePlan& plan, void* ws,
                                     hipStream_t st, int* nlaunch) {
  float* part = plan.splits > 1 ? static_cast<float*>(ws) : nullptr;
  auto go = [&](auto bmc, auto uc) {
    constexpr int BM = decltype(bmc)::value;
    const dim3 grid((unsigned)((a.N + 127) / 128), (unsigned)((a.M + BM - 1) / BM),
                    (unsigned)plan.splits);
    hipLaunchKernelGGL((glu_wide_kernel<DT, BITS, GS, BM, decltype(uc)::value>), grid, dim3(256),
                       0, st, (const uint16_t*)a.x, a.wg, (const uint16_t*)a.sg,
                       (const uint16_t*)a.bg, a.wu, (const uint16_t*)a.su, (const uint16_t*)a.bu,
                       (uint16_t*)a.out, a.gf, a.uf, part, (int)a.M, (int)a.N, (int)a.K, a.act,
                       plan.splits);
  };
  const int u = min(wide_unit(a.K, a.sg, a.bg), wide_unit(a.K, a.su, a.bu));
  auto by_u = [&](auto bmc) {
    if (u == 4) go(bmc, std::integral_constant<int, 4>{});
    else if (u == 2) go(bmc, std::integral_constant<int, 2>{});
    else go(bmc, std::integral_constant<int, 1>{});
  };
  switch (plan.bm) {
    case 64: by_u(std::integral_constant<int, 64>{}); break;
    case 128: by_u(std::integral_constant<int, 128>{}); break;
    case 192: by_u(std::integral_constant<int, 192>{}); break;
    default: by_u(std::integral_constant<int, 256>{}); break;
  }
  *nlaunch += 1;
  if (part) {
    const uint32_t quads = (uint32_t)(a.M * glu_plane(a.N) / 4);
    const bool vec = a.N % 8 == 0 && (uintptr_t)a.out % 8 == 0 &&
                     (((uintptr_t)a.gf | (uintptr_t)a.uf) & 15u) == 0;
    auto reduce = [&](auto kern) {
      hipLaunchKernelGGL(kern, dim3((quads + 255) / 256), dim3(256), 0, st, part,
                         (uint16_t*)a.out, a.gf, a.uf, quads, (int)a.N, plan.splits, a.act);
    };
    if (vec) reduce(glu_reduce_kernel<DT, true>);
    else reduce(glu_reduce_kernel<DT, false>);
    *nlaunch += 1;
  }
  return 0;
}

}  // namespace mq
