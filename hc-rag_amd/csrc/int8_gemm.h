// int8_gemm.h — the int8 product for many tokens: output tiles on an LDS-DMA ring.
//   int8_linear_tiles   a workgroup per tile (several workgroups per CU)
//   int8_linear_stream  a workgroup per CU that walks over its tiles without stopping between them
//
// A wave computes 16 MT features x 64 tokens, as MT x 4 blocks of 16x16x64 MFMAs; depth goes by in
// stages of 64 bytes per row, of which the ring holds NST, NST - 1 in flight.
//   * A DMA piece is 1 KiB of LDS: 16 rows of a stage.  The 16-byte chunks of a row are permuted on
//     the way in (the lane's global address is, the LDS image is linear), so that the fragment reads
//     of 16 rows hit every bank once.
//   * Rows past the operand's end and depth past the row's end: the descriptors end with the
//     operand's last row, rows past it only feed outputs that are not stored, and w's fragments are
//     zeroed past K in the last stage, so whatever else a stage holds is multiplied by 0.
// Host-checked: w, x and out each within 2^31 bytes (the host cuts longer batches).
#pragma once
#include <type_traits>
#include "int8_kernels.h"
#include "ring_common.h"

namespace hcr {

// 4 + 4 fragments of 16 rows each (1 KiB apart), one wait.  Inline asm: a compiler-visible LDS read
// after the loop's LDS-DMA would get a vmcnt(0) in front of it, draining the ring.
__device__ __forceinline__ void i8_read_frags(uint32_t a, uint32_t b, intx4 (&av)[4], intx4 (&bq)[4]) {
  asm volatile(
      "ds_read_b128 %0, %8\n\t"
      "ds_read_b128 %1, %8 offset:1024\n\t"
      "ds_read_b128 %2, %8 offset:2048\n\t"
      "ds_read_b128 %3, %8 offset:0xc00\n\t"
      "ds_read_b128 %4, %9\n\t"
      "ds_read_b128 %5, %9 offset:1024\n\t"
      "ds_read_b128 %6, %9 offset:2048\n\t"
      "ds_read_b128 %7, %9 offset:0xc00\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(av[0]), "=&v"(av[1]), "=&v"(av[2]), "=&v"(av[3]), "=&v"(bq[0]), "=&v"(bq[1]), "=&v"(bq[2]),
        "=&v"(bq[3])
      : "v"(a), "v"(b)
      : "memory");
}

__device__ __forceinline__ void i8_read_frags(uint32_t a, uint32_t b, intx4 (&av)[2], intx4 (&bq)[4]) {
  asm volatile(
      "ds_read_b128 %0, %6\n\t"
      "ds_read_b128 %1, %6 offset:1024\n\t"
      "ds_read_b128 %2, %7\n\t"
      "ds_read_b128 %3, %7 offset:1024\n\t"
      "ds_read_b128 %4, %7 offset:2048\n\t"
      "ds_read_b128 %5, %7 offset:0xc00\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(av[0]), "=&v"(av[1]), "=&v"(bq[0]), "=&v"(bq[1]), "=&v"(bq[2]), "=&v"(bq[3])
      : "v"(a), "v"(b)
      : "memory");
}

// 8 + 4 fragments and, while they are under way, the wave's 4 DMA pieces of a later stage (rows v, depth
// k, to lds + 0 / 8 / 16 / 24 KiB): a piece holds the wave's issue for about as long as a fragment takes
// to arrive, and before the reads the pieces would add that to the phase (8192^3: 513 us, so 476).
// (m0, where a piece goes, is a reserved register: the clobber is kept all the same)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
#define HCR_I8_DMA(V, RS, OFS)                              \
  "s_add_u32 m0, %[lds], " OFS "\n\t"                       \
  "s_nop 0\n\t"                                             \
  "buffer_load_dwordx4 %[" V "], %[" RS "], %[k] offen lds\n\t"
__device__ __forceinline__ void i8_read_frags(uint32_t a, uint32_t b, intx4 (&av)[8], intx4 (&bq)[4], intx4 wrs, intx4 xrs,
                                              const int (&v)[4], int k, uint32_t lds) {
  asm volatile(
      "ds_read_b128 %8, %[b]\n\t"
      "ds_read_b128 %9, %[b] offset:1024\n\t"
      "ds_read_b128 %10, %[b] offset:2048\n\t"
      "ds_read_b128 %11, %[b] offset:0xc00\n\t"
      "ds_read_b128 %0, %[a]\n\t"
      "ds_read_b128 %1, %[a] offset:1024\n\t"
      "ds_read_b128 %2, %[a] offset:2048\n\t"
      "ds_read_b128 %3, %[a] offset:0xc00\n\t"
      "ds_read_b128 %4, %[a] offset:4096\n\t"
      "ds_read_b128 %5, %[a] offset:5120\n\t"
      "ds_read_b128 %6, %[a] offset:6144\n\t"
      "ds_read_b128 %7, %[a] offset:7168\n\t"
      HCR_I8_DMA("v0", "wr", "0")
      HCR_I8_DMA("v1", "wr", "8192")
      HCR_I8_DMA("v2", "xr", "16384")
      HCR_I8_DMA("v3", "xr", "24576")
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(av[0]), "=&v"(av[1]), "=&v"(av[2]), "=&v"(av[3]), "=&v"(av[4]), "=&v"(av[5]), "=&v"(av[6]),
        "=&v"(av[7]), "=&v"(bq[0]), "=&v"(bq[1]), "=&v"(bq[2]), "=&v"(bq[3])
      : [a] "v"(a), [b] "v"(b), [wr] "s"(wrs), [xr] "s"(xrs), [v0] "v"(v[0]), [v1] "v"(v[1]), [v2] "v"(v[2]),
        [v3] "v"(v[3]), [k] "s"(k), [lds] "s"(lds)
      : "memory", "m0", "scc");
}
#undef HCR_I8_DMA
#pragma clang diagnostic pop
// a raw buffer descriptor for the above
__device__ __forceinline__ intx4 i8_rsrc(const void* p, int bytes) {
  const uint64_t u = (uint64_t)uniform_ptr(p);
  return intx4{(int)(uint32_t)u, (int)((uint32_t)(u >> 32) & 0xFFFFu), __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
__device__ __forceinline__ void i8_lds_read4(uint32_t a, uint32_t b, float4 (&u)[2], float4 (&v)[2]) {
  asm volatile(
      "ds_read_b128 %0, %4\n\t"
      "ds_read_b128 %1, %4 offset:64\n\t"
      "ds_read_b128 %2, %5\n\t"
      "ds_read_b128 %3, %5 offset:64\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(u[0]), "=&v"(u[1]), "=&v"(v[0]), "=&v"(v[1])
      : "v"(a), "v"(b)
      : "memory");
}
__device__ __forceinline__ void i8_lds_read_tx(uint32_t a, float (&t)[4]) {
  asm volatile(
      "ds_read_b32 %0, %4\n\t"
      "ds_read_b32 %1, %4 offset:64\n\t"
      "ds_read_b32 %2, %4 offset:128\n\t"
      "ds_read_b32 %3, %4 offset:192\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(t[0]), "=&v"(t[1]), "=&v"(t[2]), "=&v"(t[3])
      : "v"(a)
      : "memory");
}
__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rs, char* lds_dst, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (__attribute__((address_space(3))) void*)lds_dst, 4, voff, soff, 0, 0);
}

// f(integral_constant<int, 0>) .. f(integral_constant<int, N - 1>): a descriptor picked by a loop
// index rather than a constant ends up in memory and is read back lane by lane
template <int N, typename F>
__device__ __forceinline__ void i8_for(F&& f) {
  if constexpr (N > 0) {
    i8_for<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

constexpr int I8_FAR = (int)0x80000000;                // an offset past every descriptor here

__host__ __device__ constexpr int i8_size(int ot) { return ot == HCR_F32 ? 4 : 2; }

// A wave's 16 MT features x 64 tokens leave straight from the accumulators: two row blocks' 16-bit
// quads are exchanged between neighbouring 16-lane rows, after which a lane holds 8 features of a
// token and a store covers 16 tokens x 64 bytes (f32: 4 features, the same 64 bytes).  The 2 MT
// (f32: 4 MT) 16-byte buffer stores are unconditional -- what lies outside is dropped by the
// descriptor -- so that a wave issues that many for every tile; with ODD (a row is no whole number of
// 16 bytes) the features of its last, partial 16 bytes follow one by one.  (Rows need only their
// elements' alignment.)  Without the ODD code the stream kernel holds 30 registers less:
// T = 21853, N = 2304, K = 768 57 us, with it 64.
// sw, sb, sx: LDS addresses of the wave's w scales, biases and x scales.
// Measured against staging the tile through LDS for 256-byte stores, with 128 x 256 tiles of 4 waves
// at K = 768, N = 2304, T = 21853: 60.8 us, staged 62.8.
// NT: the stores are non-temporal (a result that no cache holds).
template <int OT, int MT, bool ODD, bool NT>
__device__ __forceinline__ void i8_store_tile(const I8LinearArgs& a, __amdgpu_buffer_rsrc_t o_rsrc,
                                              const intx4 (&acc)[MT][4], int lane, int f0, int t0, uint32_t sw,
                                              uint32_t sb, uint32_t sx) {
  constexpr int ES = i8_size(OT), PER = 16 / ES;       // elements per 16 bytes
  const int fr = lane & 15, fc = lane >> 4;            // accumulator: token fr, feature quad fc
  float tx[4];
  i8_lds_read_tx(sx + fr * 4, tx);
  // The whole offset in a VGPR: with one in an SGPR the compiler leaves no wait between a 16-byte
  // store and a write to its data registers, and the store took the new value in its last lanes.
  int row[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) row[n] = ((t0 + n * 16 + fr) * (int)a.ldo + f0) * ES;
  const int left = a.N - f0;                           // features that exist from f0 on
  const bool biased = a.bias != nullptr;
#pragma unroll
  for (int p = 0; p < MT / 2; ++p) {
    float4 s4[2], b4[2];
    i8_lds_read4(sw + (p * 32 + fc * 4) * 4, sb + (p * 32 + fc * 4) * 4, s4, b4);
#pragma unroll
    for (int mi = 0; mi < 2; ++mi)
      if (!biased) b4[mi] = float4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      float v[2][4];
#pragma unroll
      for (int mi = 0; mi < 2; ++mi) {
        const intx4 c = acc[2 * p + mi][n];
        v[mi][0] = fmaf((float)c[0] * tx[n], s4[mi].x, b4[mi].x);
        v[mi][1] = fmaf((float)c[1] * tx[n], s4[mi].y, b4[mi].y);
        v[mi][2] = fmaf((float)c[2] * tx[n], s4[mi].z, b4[mi].z);
        v[mi][3] = fmaf((float)c[3] * tx[n], s4[mi].w, b4[mi].w);
      }
      constexpr int NU = OT == HCR_F32 ? 2 : 1;
      uintx4 u[NU];
      int f[NU];
      if constexpr (OT == HCR_F32) {
#pragma unroll
        for (int mi = 0; mi < 2; ++mi) {
          f[mi] = p * 32 + mi * 16 + fc * 4;
          u[mi] = uintx4{__float_as_uint(v[mi][0]), __float_as_uint(v[mi][1]), __float_as_uint(v[mi][2]),
                         __float_as_uint(v[mi][3])};
        }
      } else {
        using H = typename std::conditional<OT == HCR_BF16, __bf16, _Float16>::type;
        // the 16-lane rows 0..3 hold quads fc of block 0 in x and of block 1 in y; after the swap an
        // even row holds quads fc, fc + 1 of block 0, an odd row fc - 1, fc of block 1
        const auto lo = __builtin_amdgcn_permlane16_swap(i8_pack2<H>(v[0][0], v[0][1]), i8_pack2<H>(v[1][0], v[1][1]), false, false);
        const auto hi = __builtin_amdgcn_permlane16_swap(i8_pack2<H>(v[0][2], v[0][3]), i8_pack2<H>(v[1][2], v[1][3]), false, false);
        f[0] = p * 32 + (fc & 1) * 16 + (fc >> 1) * 8;
        u[0] = uintx4{lo[0], hi[0], lo[1], hi[1]};
      }
#pragma unroll
      for (int j = 0; j < NU; ++j) {
        __builtin_amdgcn_raw_buffer_store_b128(u[j], o_rsrc, f[j] + PER <= left ? row[n] + f[j] * ES : I8_FAR, 0, NT ? 2 : 0);
        if (ODD && left < 16 * MT) {                   // (uniform: the wave holds the row's last features)
          const uint32_t w[4] = {u[j][0], u[j][1], u[j][2], u[j][3]};
#pragma unroll
          for (int e = 0; e < PER - 1; ++e) {
            const int at = f[j] < left && f[j] + PER > left && f[j] + e < left ? row[n] + (f[j] + e) * ES : I8_FAR;
            if constexpr (OT == HCR_F32) __builtin_amdgcn_raw_buffer_store_b32(w[e], o_rsrc, at, 0, 0);
            else __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(w[e >> 1] >> (16 * (e & 1))), o_rsrc, at, 0, 0);
          }
        }
      }
    }
  }
}

// A workgroup of WM x WN waves per tile of 16 MT WM features x 64 WN tokens; OCC waves per SIMD, so that
// while one workgroup of a CU waits for its stage or stores its tile another multiplies.
template <int OT, bool ODD, int MT, int WM, int WN, int NST, int OCC, bool NT>
__global__ void __launch_bounds__(64 * WM * WN, OCC)
int8_linear_tiles(I8LinearArgs a, int n_tiles_feat) {
  constexpr int KB = 64, FT = 16 * MT * WM, TT = 64 * WN, NW = WM * WN;
  constexpr int NA = FT / 16 / NW, NB = TT / 16 / NW;  // W and X pieces per wave and stage
  constexpr int A_BYTES = FT * KB, STAGE = (FT + TT) * KB, D = NST - 1, NPC = NA + NB;
  __shared__ __attribute__((aligned(16))) char ring[NST * STAGE];
  __shared__ __attribute__((aligned(16))) float sc[2 * FT + TT];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  // consecutive g share the token tile and run on one XCD (workgroups go round the 8 XCDs)
  const unsigned nwg = gridDim.x, b = blockIdx.x;
  const unsigned xcd = b & 7, q8 = nwg >> 3, r8 = nwg & 7;
  const unsigned g = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (b >> 3);
  const int f0 = (int)(g % (unsigned)n_tiles_feat) * FT, t0 = (int)(g / (unsigned)n_tiles_feat) * TT;

  for (int i = tid; i < FT; i += 64 * NW) {
    const int f = min(f0 + i, a.N - 1);
    sc[i] = a.sw[f];
    sc[FT + i] = a.bias ? a.bias[f] : 0.f;
  }
  for (int i = tid; i < TT; i += 64 * NW) sc[2 * FT + i] = a.sx[min(t0 + i, a.T - 1)];

  const int kend = (a.K + 15) & ~15;                   // (a row's last chunk is inside its stride)
  const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      uniform_ptr(a.w), (short)0, (a.N - 1) * (int)a.ldw + kend, 0x00020000);
  const __amdgpu_buffer_rsrc_t x_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      uniform_ptr(a.x), (short)0, (a.T - 1) * (int)a.ldx + kend, 0x00020000);
  const int drow = lane >> 2;
  const int dchunk = (lane & 3) ^ (int)((V3_SWZ >> (((lane >> 4) & 3) * 4)) & 3u);
  // A piece's offset of rows is in the lane's part, only the depth (below the operand's size) in the
  // scalar part: a range check compares the first with the size less the second.
  int voff[NPC];
#pragma unroll
  for (int i = 0; i < NA; ++i) voff[i] = (f0 + (wave + NW * i) * 16 + drow) * (int)a.ldw + dchunk * 16;
#pragma unroll
  for (int i = 0; i < NB; ++i) voff[NA + i] = (t0 + (wave + NW * i) * 16 + drow) * (int)a.ldx + dchunk * 16;
  const int nsteps = (a.K + KB - 1) / KB;
  int is_s = 0, is_slot = 0;
  auto issue = [&](auto piece) __attribute__((always_inline)) {
    constexpr int i = decltype(piece)::value;
    // (past the last stage the pieces are still issued, for the waits' counts, but read nothing)
    const bool live = is_s < nsteps;
    const int far = __builtin_amdgcn_readfirstlane(live ? 0 : I8_FAR);
    const int kofs = __builtin_amdgcn_readfirstlane(live ? is_s * KB : 0);
    char* st = ring + __builtin_amdgcn_readfirstlane(is_slot) * STAGE;
    if constexpr (i < NA) dma16(w_rsrc, st + (wave + NW * i) * 1024, voff[i] | far, kofs);
    else dma16(x_rsrc, st + A_BYTES + (wave + NW * (i - NA)) * 1024, voff[i] | far, kofs);
  };
  auto advance = [&]() __attribute__((always_inline)) {
    ++is_s;
    is_slot = (is_slot + 1 == NST) ? 0 : is_slot + 1;
  };
  for (int i = 0; i < D; ++i) {
    i8_for<NPC>(issue);
    advance();
  }

  const int fr = lane & 15, fc = lane >> 4;
  const int slot = v3_slot(fc, fr);
  const int offA = (wm * 16 * MT + fr) * KB + slot * 16;
  const int offB = A_BYTES + (wn * 64 + fr) * KB + slot * 16;
  intx4 acc[MT][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = intx4{0, 0, 0, 0};

  int rslot = 0;
  for (int s = 0; s < nsteps; ++s) {
    v3_wait_vmcnt((D - 1) * NPC);
    v3_barrier();
    const char* st = ring + rslot * STAGE;
    intx4 av[MT], bq[4];
    i8_read_frags(lds_addr(st + offA), lds_addr(st + offB), av, bq);
    if ((s + 1) * KB > a.K) {
      const int n = a.K - s * KB - fc * 16;
#pragma unroll
      for (int m = 0; m < MT; ++m) av[m] = i8_keep(av[m], n);
    }
    i8_for<MT>([&](auto mc) __attribute__((always_inline)) {
      constexpr int m = decltype(mc)::value;
#pragma unroll
      for (int n = 0; n < 4; ++n) acc[m][n] = i8_mfma(av[m], bq[n], acc[m][n]);
      i8_for<NPC>([&](auto kc) __attribute__((always_inline)) {    // the pieces spread over the MFMAs
        if constexpr (decltype(kc)::value * MT / NPC == m) issue(kc);
      });
    });
    advance();
    rslot = (rslot + 1 == NST) ? 0 : rslot + 1;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // the ring's last pieces, before the LDS is given back
  const __amdgpu_buffer_rsrc_t o_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      uniform_ptr(a.out), (short)0, __builtin_amdgcn_readfirstlane(((a.T - 1) * (int)a.ldo + a.N) * i8_size(OT)), 0x00020000);
  i8_store_tile<OT, MT, ODD, NT>(a, o_rsrc, acc, lane, f0 + wm * 16 * MT, t0 + wn * 64, lds_addr(sc + wm * 16 * MT),
                             lds_addr(sc + FT + wm * 16 * MT), lds_addr(sc + 2 * FT + wn * 64));
}

// -------------------------------------------------------------------------------------
// Many tiles: one workgroup per CU walks over its output tiles (256 features x 256 tokens, 8
// waves) as one stream of 64-byte stages that does not stop at a tile's end: the LDS-DMA runs 3
// stages ahead into the next tile, and a tile's stores drain under the next one's stages.
//   * The waves form two groups (one wave of each per SIMD) half a stage apart: while a group reads
//     its fragments (R) the other runs its 32 MFMAs (M), with a barrier between phases, so that the
//     matrix cores do not wait for LDS and the fragment reads do not collide.
//   * Phases: group 0 has R(s) in phase 2s and M(s) in 2s + 1, group 1 one later.  Stage s + 3 goes
//     to the slot of stage s - 1, whose last reads (group 1's R(s - 1)) end with phase 2s - 1; both
//     groups issue it in their R(s).  Before phase 2s every wave has waited for its own pieces of
//     stage s.
//   * Every wave issues at least NS stores per tile (i8_store_tile), which the vmcnt waits rely on: a
//     wait for stage s + 1 may leave the pieces of s + 2 and s + 3 and, in a tile's first two
//     stages, NS of the previous tile's stores (issued between the pieces of its s + 2 and s + 3),
//     which are newer than the stage waited for.
//   * The tile's scales and biases come with its stage 0, into one of 4 buffers (the stream is up to
//     4 stages ahead of group 1's epilogue: at 2 stages a tile, 2 tiles).
// Host-checked: K > 64 (2 stages a tile at least).
// OT: hcr_dtype of out
template <int OT, bool ODD, bool NT>
__global__ void __launch_bounds__(512, 2)
int8_linear_stream(I8LinearArgs a, int n_tiles_feat, unsigned n_tiles) {
  constexpr int KB = 64, NST = 4, FT = 256, TT = 256, A_BYTES = FT * KB, STAGE = (FT + TT) * KB;
  constexpr int NS = OT == HCR_F32 ? 32 : 16;          // stores per wave and tile
  constexpr int SC = 2 * FT + TT;
  __shared__ __attribute__((aligned(16))) char ring[NST * STAGE];
  __shared__ __attribute__((aligned(16))) float sc[4][SC];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3, grp = wave >> 2;
  // XCD x (workgroups go round the 8 XCDs) takes a contiguous run of tiles, its workgroups side by
  // side: at any time an XCD works on few token tiles, whose rows and the weights sit in its L2
  const unsigned xcd = blockIdx.x & 7, per = gridDim.x >> 3;   // (host: a multiple of 8 workgroups)
  const unsigned q8 = n_tiles >> 3, r8 = n_tiles & 7;
  const unsigned first = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8);
  const unsigned many = xcd < r8 ? q8 + 1 : q8, mine = blockIdx.x >> 3;
  if (mine >= many) return;
  const int my_tiles = (int)((many - mine + per - 1) / per);

  const int kend = (a.K + 15) & ~15;
  const __amdgpu_buffer_rsrc_t w_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      uniform_ptr(a.w), (short)0, (a.N - 1) * (int)a.ldw + kend, 0x00020000);
  const __amdgpu_buffer_rsrc_t x_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      uniform_ptr(a.x), (short)0, (a.T - 1) * (int)a.ldx + kend, 0x00020000);
  const __amdgpu_buffer_rsrc_t sx_rsrc = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(a.sx), (short)0, a.T * 4, 0x00020000);
  // (waves 0-3 bring the w scales, 4-7 the biases)
  const float* fsrc = (wave < 4 || !a.bias) ? a.sw : a.bias;
  const __amdgpu_buffer_rsrc_t f_rsrc = __builtin_amdgcn_make_buffer_rsrc(uniform_ptr(fsrc), (short)0, a.N * 4, 0x00020000);
  const __amdgpu_buffer_rsrc_t o_rsrc = __builtin_amdgcn_make_buffer_rsrc(
      uniform_ptr(a.out), (short)0, ((a.T - 1) * (int)a.ldo + a.N) * i8_size(OT), 0x00020000);

  const int drow = lane >> 2;
  const int dchunk = (lane & 3) ^ (int)((V3_SWZ >> (((lane >> 4) & 3) * 4)) & 3u);
  const int nsteps = (a.K + KB - 1) / KB;
  auto tile_at = [&](int i, int& f0, int& t0) __attribute__((always_inline)) {
    const unsigned g = first + mine + (unsigned)i * per;
    f0 = __builtin_amdgcn_readfirstlane((int)(g % (unsigned)n_tiles_feat) * FT);
    t0 = __builtin_amdgcn_readfirstlane((int)(g / (unsigned)n_tiles_feat) * TT);
  };
  // the stream's head: stage is_s of tile is_i, bound for slot is_slot
  int is_s = 0, is_i = 0, is_slot = 0;
  int voff[4];                                         // (rows here, the depth in the scalar part: see above)
  auto stage_rows = [&]() __attribute__((always_inline)) {
    const bool live = is_i < my_tiles;
    if (live && is_s == 0) {
      int f0, t0;
      tile_at(is_i, f0, t0);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = (wave + 8 * i) * 16 + drow;
        voff[i] = (f0 + r) * (int)a.ldw + dchunk * 16;
        voff[2 + i] = (t0 + r) * (int)a.ldx + dchunk * 16;
      }
      char* s = reinterpret_cast<char*>(sc[is_i & 3]);
      dma4(f_rsrc, s + wave * 256, (f0 + (wave & 3) * 64 + lane) * 4, 0);
      if (wave < 4) dma4(sx_rsrc, s + 2 * FT * 4 + wave * 256, (t0 + wave * 64 + lane) * 4, 0);
    }
  };
  auto stage_next = [&]() __attribute__((always_inline)) {
    is_slot = (is_slot + 1) & (NST - 1);
    if (++is_s == nsteps) { is_s = 0; ++is_i; }
  };

  const int fr = lane & 15, fc = lane >> 4;            // (accumulator: token fr, feature quad fc)
  const int slot = v3_slot(fc, fr);
  const int offA = (wm * 128 + fr) * KB + slot * 16;
  const int offB = A_BYTES + (wn * 64 + fr) * KB + slot * 16;
  intx4 acc[8][4];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int m = 0; m < 8; ++m)
#pragma unroll
      for (int n = 0; n < 4; ++n) acc[m][n] = intx4{0, 0, 0, 0};
  };
  auto store_tile = [&](int i) __attribute__((always_inline)) {
    int f0, t0;
    tile_at(i, f0, t0);
    const uint32_t s0 = lds_addr(sc[i & 3]);
    i8_store_tile<OT, 8, ODD, NT>(a, o_rsrc, acc, lane, f0 + wm * 128, t0 + wn * 64, s0 + wm * 512,
                              s0 + (FT + wm * 128) * 4, s0 + (2 * FT + wn * 64) * 4);
  };

  for (int i = 0; i < NST - 1; ++i) {
    stage_rows();
    const int far = __builtin_amdgcn_readfirstlane(is_i < my_tiles ? 0 : I8_FAR);
    const int kofs = __builtin_amdgcn_readfirstlane(is_i < my_tiles ? is_s * KB : 0);
    char* st = ring + __builtin_amdgcn_readfirstlane(is_slot) * STAGE;
    dma16(w_rsrc, st + wave * 1024, voff[0] | far, kofs);
    dma16(w_rsrc, st + (wave + 8) * 1024, voff[1] | far, kofs);
    dma16(x_rsrc, st + A_BYTES + wave * 1024, voff[2] | far, kofs);
    dma16(x_rsrc, st + A_BYTES + (wave + 8) * 1024, voff[3] | far, kofs);
    stage_next();
  }
  const intx4 wrs = i8_rsrc(a.w, (a.N - 1) * (int)a.ldw + kend), xrs = i8_rsrc(a.x, (a.T - 1) * (int)a.ldx + kend);
  clear();
  v3_wait_vmcnt(8);
  v3_barrier();
  if (grp) v3_barrier();
  int rslot = 0;
  for (int ti = 0; ti < my_tiles; ++ti) {
    for (int s = 0; s < nsteps; ++s) {
      stage_rows();
      __builtin_amdgcn_sched_barrier(0);
      if (s == 0 && ti) {
        store_tile(ti - 1);
        clear();
      }
      __builtin_amdgcn_sched_barrier(0);
      const char* st = ring + rslot * STAGE;
      intx4 av[8], bq[4];
      // (past the last tile the pieces are still issued, for the waits' counts, but read nothing)
      const bool live = is_i < my_tiles;
      const int far = __builtin_amdgcn_readfirstlane(live ? 0 : I8_FAR);
      const int vo[4] = {voff[0] | far, voff[1] | far, voff[2] | far, voff[3] | far};
      i8_read_frags(lds_addr(st + offA), lds_addr(st + offB), av, bq, wrs, xrs, vo,
                    __builtin_amdgcn_readfirstlane(live ? is_s * KB : 0),
                    __builtin_amdgcn_readfirstlane(lds_addr(ring) + is_slot * STAGE + wave * 1024));
      stage_next();
      if ((s + 1) * KB > a.K) {
        const int n = a.K - s * KB - fc * 16;
#pragma unroll
        for (int m = 0; m < 8; ++m) av[m] = i8_keep(av[m], n);
      }
      const bool stores = ti && s < 2;                 // the previous tile's are newer than stage s + 1
      if (grp) { if (stores) v3_wait_vmcnt(8 + NS); else v3_wait_vmcnt(8); }
      v3_barrier();
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int m = 0; m < 8; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) acc[m][n] = i8_mfma(av[m], bq[n], acc[m][n]);
      __builtin_amdgcn_s_setprio(0);
      __builtin_amdgcn_sched_barrier(0);
      if (!grp) { if (stores) v3_wait_vmcnt(8 + NS); else v3_wait_vmcnt(8); }
      v3_barrier();
      rslot = (rslot + 1) & (NST - 1);
    }
  }
  if (!grp) v3_barrier();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // the ring's last pieces, before the LDS is given back
  store_tile(my_tiles - 1);
}

}  // namespace hcr
