// The tiled product of block-scaled e4m3 rows with e4m3 weights, shared by the linear and the experts:
//   y[m, n] = sum_b sx[m, b] sw[n / 128, b] sum_{k in block b} qx[m, k] qw[n, k].
//
// A workgroup owns BN weight rows x BM activation rows; a step is one block of 128 columns, whose tiles (128
// bytes a row) go from memory straight to LDS while the step before is multiplied. The 16-byte pieces of a
// row are stored rotated by the pair of rows it is of (f8_slot), so that the fragments' 16-byte reads meet no bank twice; the
// rotation is done on the global side of the load, whose LDS side is linear by construction. The MFMAs
// take the weights as A, so a lane holds one activation row's outputs: both scales are one factor a lane and step, and
// the fp32 sum over blocks is one fma per output and step beside 128 products of the matrix cores.
//
// MODE 0: y bf16 [M, N], or fp32 partials of a K range.
// MODE 1: the experts' gate_up: rows sorted by expert, tile rows [0, BN/2) gate and [BN/2, BN) up of the same
//         128 columns of h; the epilogue forms h = silu(g) u in fp32 and quantizes it. Products by the bf16 instruction
//         (f8_widen), as h's codes hang on them: 4096 tokens of 8 of 64 experts of 2048 x 1024 take 526 us, 426 by
//         the e4m3 one.
// MODE 2: the experts' down: rows sorted by expert, written back in routed order, in fp32.
#pragma once

#include "f8_common.h"

namespace imq {

struct F8Tile {
  const uint8_t* x;      // e4m3 rows, row stride sx bytes
  int64_t sx;
  const float* xs;       // scale of row m, block b at m * xsm + b * xsb
  int64_t xsm, xsb;
  const uint8_t* w;      // e4m3 weight rows
  int64_t sw, swe;       // row and expert stride in bytes
  const float* ws;       // scale of row block r, block b (expert e) at e * wse + r * wsr + b * wsb
  int64_t wsr, wsb, wse;
  int M, N, nb;          // nb: blocks of 128 columns
  uint16_t* y;
  int64_t sy;
  float* rows;           // MODE 2: routed row m, fp32, at m * sy
  float* part;           // MODE 0, fp32 partials [splits][M][N] when splits > 1
  int splits;
  int mt, nt;            // tiles along M (MODE 0) and N
  // experts
  const int32_t* tiles;  // tiles[0]: number of row tiles; then {expert, first sorted row, end} each
  const int32_t* perm;   // sorted position -> routed row
  FastDiv kd;            // MODE 1: x row = routed row / k
  int I;
  uint8_t* h;            // MODE 1 out: e4m3 [B][sh], scales [I blocks][hsb]
  int64_t sh;
  float* hs;
  int64_t hsb;
};

}  // namespace imq

namespace {

using imq::F8Tile;

// 16 bytes a lane from base + off + soff to LDS at lds + 16 lane (lds wave-uniform). The destination register is M0 and no
// other register is written, so nothing can be reused while the load is in flight; the kernel waits with
// s_waitcnt vmcnt before the barrier that lets the tile be read.
IMQ_DEV void f8_to_lds(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds" ::"v"(off), "s"(r), "s"(lds), "s"(soff)
               : "memory", "m0");
}

// The same with 4 bytes a lane.
IMQ_DEV void f8_to_lds4(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t soff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %3 offen lds" ::"v"(off), "s"(r), "s"(lds), "s"(soff)
               : "memory", "m0");
}

IMQ_DEV __amdgpu_buffer_rsrc_t f8_rsrc(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, 0x7fffffff, 0x00020000);
}

IMQ_DEV uint32_t f8_lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

// Where piece p of tile row `row` lies in the row: the 64 banks hold two rows, so 16 lanes that read the same piece of 16
// consecutive rows meet each bank once if rows 2 i and 2 i + 1 rotate alike (rotated by row % 8, rows 8 apart met in the
// same banks, and half of the LDS time was conflicts).
IMQ_DEV int f8_slot(int row, int p) { return p ^ ((row >> 1) & 7); }

// The lane's 32 bytes of tile row `row` (a step's 128 columns): pieces 2 g and 2 g + 1 of lane group g = lane / 16.
IMQ_DEV i32x8_t f8_frag(const uint8_t* tile, int row, int g) {
  const u32x4_t lo = *(const u32x4_t*)(tile + row * 128 + (f8_slot(row, 2 * g) << 4));
  const u32x4_t hi = *(const u32x4_t*)(tile + row * 128 + (f8_slot(row, 2 * g + 1) << 4));
  return f8_join(lo, hi);
}

// Bytes of a buffer: weight rows, activation rows, a scale per activation row.
constexpr int f8_stage_bytes(int BN, int BM) { return (BN + BM) * 128 + (BM < 64 ? 64 : BM) * 4; }

// A tile's results. Those in bf16 and h's codes go through `lds` (the last step's buffer; 16-byte pieces rotated by the row, as the operands'),
// so that memory sees whole rows of the tile: a lane holds 4 columns of one row, and storing those 8 bytes at a time cost
// as much as 30 steps. Waits for the wave's loads before its first store.
template <int BN, int BM, int WN, int WM, int MODE, typename ACC>
IMQ_DEV void f8_epilogue(const F8Tile& a, int m0, int mend, int n0, int split, uint8_t* lds, ACC& acc) {
  constexpr int W = WN * WM, TN = BN / WN, TM = BM / WM, IN = TN / 16, IM = TM / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN, c = lane & 15, g = lane >> 4;
  if constexpr (MODE == 0) {
    if (a.splits > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int j = 0; j < IM; ++j) {
        const int m = m0 + wm * TM + j * 16 + c;
        if (m >= mend) continue;
        float* p = a.part + ((int64_t)split * a.M + m) * a.N;
#pragma unroll
        for (int i = 0; i < IN; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int n = n0 + wn * TN + i * 16 + 4 * g + r;
            if (n < a.N) p[n] = acc[i][j][r];
          }
      }
      return;
    }
  }
  if constexpr (MODE == 2) {
    // A routed row stays fp32 until the combine has summed its token's: a column may be as far below its neighbours as it
    // likes, and one that is not finite spoils no other. Straight from the registers: a lane's 4 columns are 16 bytes, a
    // row's four lane groups 64 on end.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
    for (int j = 0; j < IM; ++j) {
      const int m = m0 + wm * TM + j * 16 + c;
      if (m >= mend) continue;
      float* y = a.rows + (int64_t)a.perm[m] * a.sy + n0 + wn * TN + 4 * g;
#pragma unroll
      for (int i = 0; i < IN; ++i)
        if (n0 + wn * TN + i * 16 + 4 * g < a.N) *(f32x4_t*)(y + i * 16) = acc[i][j];     // the stride is whole fours, past N slack
    }
  } else if constexpr (MODE == 0) {
    constexpr int PC = BN / 8;                           // pieces of 8 columns a row
    // the buffer holds BM / PASSES rows at a time
    constexpr int PASSES = BM * BN * 2 > (BN + BM) * 128 ? 2 : 1, ROWS = BM / PASSES;
    static_assert(BM % PASSES == 0 && WM % PASSES == 0, "whole waves' rows a pass");
    const bool vec = (a.sy & 7) == 0 && ((uintptr_t)a.y & 15) == 0;
    lds_barrier();
#pragma unroll
    for (int s = 0; s < PASSES; ++s) {
      if (s > 0) lds_barrier();
      if (wm / (WM / PASSES) == s) {
#pragma unroll
        for (int j = 0; j < IM; ++j) {
          const int row = wm * TM + j * 16 + c;
          const int at = row - s * ROWS;
#pragma unroll
          for (int i = 0; i < IN; ++i) {
            const int piece = (wn * TN + i * 16) / 8 + (g >> 1);
            const u32x2_t w = {cvt_pk_bf16(acc[i][j][0], acc[i][j][1]), cvt_pk_bf16(acc[i][j][2], acc[i][j][3])};
            *(u32x2_t*)(lds + at * (BN * 2) + ((piece ^ (at & (PC - 1))) << 4) + 8 * (g & 1)) = w;
          }
        }
      }
      if (s == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      lds_barrier();
#pragma unroll 4
      for (int id = tid; id < ROWS * PC; id += 64 * W) {
        const int at = id / PC, piece = id % PC, n = n0 + piece * 8;
        const int64_t m = m0 + s * ROWS + at;
        if (m >= mend || n >= a.N) continue;
        const u32x4_t v = *(const u32x4_t*)(lds + at * (BN * 2) + ((piece ^ (at & (PC - 1))) << 4));
        uint16_t* y = a.y + m * a.sy + n;
        if (vec && n + 8 <= a.N) {
          *(u32x4_t*)y = v;
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint32_t w = v[q >> 1];
            if (n + q < a.N) y[q] = (uint16_t)(q & 1 ? w >> 16 : w);
          }
        }
      }
    }
  } else {
    // h = silu(g) u of 128 columns (zero past I): the block's largest magnitude over the workgroup's waves, then codes
    uint32_t* most = (uint32_t*)(lds + BM * 128);     // [WN][BM]
    lds_barrier();
#pragma unroll
    for (int j = 0; j < IM; ++j) {
      uint32_t mx = 0;
#pragma unroll
      for (int i = 0; i < IN / 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int col = n0 + wn * (TN / 2) + i * 16 + 4 * g + r;
          const float gv = acc[i][j][r], uv = acc[IN / 2 + i][j][r];
          const float v = col < a.I ? f8_silu_mul(gv, uv) : 0.f;
          acc[i][j][r] = v;
          const uint32_t bits = __float_as_uint(v) & 0x7fffffffu;
          mx = bits > mx ? bits : mx;
        }
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) {
        const uint32_t q = (uint32_t)__shfl_xor((int)mx, o, 64);
        mx = q > mx ? q : mx;
      }
      if (g == 0) most[wn * BM + wm * TM + j * 16 + c] = mx;
    }
    lds_barrier();
#pragma unroll
    for (int j = 0; j < IM; ++j) {
      const int row = wm * TM + j * 16 + c, m = m0 + row;
      uint32_t mx = 0;
#pragma unroll
      for (int q = 0; q < WN; ++q) {
        const uint32_t o = most[q * BM + row];
        mx = o > mx ? o : mx;
      }
      const float s = f8_scale(mx), rs = 1.f / s;
#pragma unroll
      for (int i = 0; i < IN / 2; ++i) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = acc[i][j][q];
        const int piece = (wn * (TN / 2)) / 16 + i;
        *(uint32_t*)(lds + row * 128 + (f8_slot(row, piece) << 4) + 4 * g) = f8_codes4(v, s, rs);
      }
      if (wn == 0 && g == 0 && m < mend) a.hs[(int64_t)(n0 / 128) * a.hsb + m] = s;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    for (int id = tid; id < BM * 8; id += 64 * W) {
      const int row = id >> 3, piece = id & 7;
      if (m0 + row >= mend) continue;
      *(u32x4_t*)(a.h + (int64_t)(m0 + row) * a.sh + n0 + piece * 16) =
          *(const u32x4_t*)(lds + row * 128 + (f8_slot(row, piece) << 4));
    }
  }
}

// S buffers of a step each; WN x WM waves. A wave computes (BN / WN) x (BM / WM) in 16 x 16 blocks, one MFMA over a step's 128 columns each.
// MODE 1 takes half of a wave's rows from the gate and half from the up rows of the same columns.
//
// With two buffers a workgroup runs one tile after the other: the loads of a tile's first step go out during the last
// step of the tile before, so its epilogue (which uses the other buffer) hides their latency and that of the row
// lookups. With more, a workgroup has one tile.
template <int BN, int BM, int WN, int WM, int S, int MODE>
__global__ __launch_bounds__(64 * WN * WM, 2) void f8_tile_kernel(F8Tile a) {
  constexpr bool WIDE = MODE == 1;
  constexpr int W = WN * WM, TN = BN / WN, TM = BM / WM, IN = TN / 16, IM = TM / 16;
  constexpr int LA = BN / 8 / W, LB = BM / 8 / W, LW = LA + LB;    // a wave's loads (8 rows of 128 bytes each) a step
  static_assert(LA * W * 8 == BN && LB * W * 8 == BM && TN % 32 == 0 && TM % 16 == 0, "tile");
  static_assert(MODE == 1 ? BN == 256 : TN <= 128 && 128 % TN == 0, "a wave's rows share a scale");
  constexpr int BYTES = f8_stage_bytes(BN, BM), XS = (BM + 63) / 64;
  extern __shared__ __attribute__((aligned(16))) uint8_t f8_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave % WN, wm = wave / WN, c = lane & 15, g = lane >> 4;
  const int row8 = lane >> 3;
  auto piece16 = [&](int row) { return f8_slot(row, lane & 7) * 16; };

  // Tiles are dealt to the XCDs (dispatch index % 8) in contiguous runs, so that the rows and weights that
  // neighbouring tiles share stay in that XCD's L2; an XCD's workgroups take its run in turn.
  const int total = MODE == 0 ? a.mt * a.nt * a.splits : __builtin_amdgcn_readfirstlane(a.tiles[0]) * a.nt;
  const int xcd = blockIdx.x % 8, q8 = total / 8, r8 = total % 8;
  const int tend = xcd < r8 ? (xcd + 1) * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8 + 1) * q8;
  const int tstep = gridDim.x / 8;
  int t = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + blockIdx.x / 8;
  if (t >= tend) return;

  struct Tile {
    int e, m0, mend, n0, split, b0, b1;
  };
  auto tile_of = [&](int t) {
    Tile v{};
    v.b1 = a.nb;
    if constexpr (MODE == 0) {
      const int T = a.mt * a.nt;
      if (a.splits > 1) {
        v.split = t / T;
        t -= v.split * T;
        v.b0 = (int)((int64_t)a.nb * v.split / a.splits);
        v.b1 = (int)((int64_t)a.nb * (v.split + 1) / a.splits);
      }
      // groups of 8 row tiles
      const int grp = t / (8 * a.nt), first = grp * 8, rows = a.mt - first < 8 ? a.mt - first : 8, in = t - grp * 8 * a.nt;
      v.m0 = (first + in % rows) * BM;
      v.n0 = (in / rows) * BN;
      v.mend = a.M;
    } else {
      const int rt = t / a.nt;
      v.e = __builtin_amdgcn_readfirstlane(a.tiles[1 + 3 * rt]);
      v.m0 = __builtin_amdgcn_readfirstlane(a.tiles[2 + 3 * rt]);
      v.mend = __builtin_amdgcn_readfirstlane(a.tiles[3 + 3 * rt]);
      v.n0 = (t - rt * a.nt) * (MODE == 1 ? BN / 2 : BN);
    }
    return v;
  };
  // Tile row r's activation row; rows past the end repeat the last one (their outputs are not stored).
  auto row_at = [&](const Tile& v, int r) {
    const int m = v.m0 + r < v.mend ? v.m0 + r : v.mend - 1;
    return MODE == 1 ? (int)div_fast((uint32_t)a.perm[m], a.kd) : m;
  };
  // MODE 1 looks rows up in memory. A workgroup of eight waves, alone on its CU, has each thread fetch one row of the
  // next tile a tile ahead and pass it on through LDS; smaller ones cover for each other.
  constexpr bool AHEAD = MODE == 1 && W == 8;
  int32_t* rows = (int32_t*)(f8_lds + S * BYTES);
  int row1 = 0;
  uint32_t off[LW], soff = 0;
  __amdgpu_buffer_rsrc_t rw, rx;
  const __amdgpu_buffer_rsrc_t rs = f8_rsrc(a.xs);
  typedef const __attribute__((address_space(4))) float cfloat;     // uniform: scalar loads
  cfloat* wsp[2];
  auto aim = [&](const Tile& v, bool ahead) {
    auto at = [&](int r) { return AHEAD && ahead ? rows[r] : row_at(v, r); };
    rw = f8_rsrc(a.w + (int64_t)v.e * a.swe + (MODE == 0 ? (int64_t)v.n0 * a.sw : 0));
    rx = f8_rsrc(a.x + (MODE == 0 ? (int64_t)v.m0 * a.sx : 0));
#pragma unroll
    for (int i = 0; i < LA; ++i) {
      const int trow = (wave * LA + i) * 8 + row8;
      int row = trow;
      if constexpr (MODE == 1) {
        const int j = v.n0 + (row < BN / 2 ? row : row - BN / 2);
        row = (j < a.I ? j : a.I - 1) + (row < BN / 2 ? 0 : a.I);
      } else if constexpr (MODE == 2) {
        row = v.n0 + row < a.N ? v.n0 + row : a.N - 1;
      } else {
        row = v.n0 + row < a.N ? row : a.N - 1 - v.n0;
      }
      off[i] = (uint32_t)row * (uint32_t)a.sw + piece16(trow);
    }
#pragma unroll
    for (int i = 0; i < LB; ++i) {
      const int trow = (wave * LB + i) * 8 + row8, row = at(trow) - (MODE == 0 ? v.m0 : 0);
      off[LA + i] = (uint32_t)row * (uint32_t)a.sx + piece16(trow);
    }
    if (wave < XS) soff = (uint32_t)at(wave * 64 + lane < BM ? wave * 64 + lane : BM - 1) * (uint32_t)a.xsm * 4u;
    const int n = v.n0 + (MODE == 1 ? 0 : wn * TN);
    wsp[0] = (cfloat*)(a.ws + (int64_t)v.e * a.wse + (int64_t)((n < a.N ? n : a.N - 1) / 128) * a.wsr);
    if constexpr (MODE == 1) wsp[1] = wsp[0] + (int64_t)((a.I + 127) / 128) * a.wsr;
  };
  const uint32_t lds0 = f8_lds_addr(f8_lds);
  auto load = [&](int b, int buf, int i) {
    if (i < LA) f8_to_lds(rw, off[i], (uint32_t)b * 128u, lds0 + buf * BYTES + (wave * LA + i) * 1024);
    else f8_to_lds(rx, off[i], (uint32_t)b * 128u, lds0 + buf * BYTES + BN * 128 + (wave * LB + i - LA) * 1024);
  };
  float wc[2];
  auto scales = [&](int b, int buf) {
    if (wave < XS) f8_to_lds4(rs, soff, (uint32_t)b * (uint32_t)a.xsb * 4u, lds0 + buf * BYTES + (BN + BM) * 128 + wave * 256);
  };
  auto wscales = [&](int b) {
    wc[0] = wsp[0][b * a.wsb];
    if constexpr (MODE == 1) wc[1] = wsp[1][b * a.wsb];
  };
  auto spread = [](int i) constexpr { return 2 * i * LW / IN < LW ? 2 * i * LW / IN : LW; };

  Tile cur = tile_of(t);
  aim(cur, false);
#pragma unroll
  for (int q = 0; q < S - 1; ++q) {
    const int b = cur.b0 + q < cur.b1 ? cur.b0 + q : cur.b1 - 1;
    scales(b, q);
#pragma unroll
    for (int i = 0; i < LW; ++i) load(b, q, i);
  }
  wscales(cur.b0);
  if constexpr (S == 2) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  int buf = 0;
  while (true) {
    t += tstep;
    const bool more = S == 2 && t < tend;
    Tile nxt = cur;
    if (more) {
      nxt = tile_of(t);
      if (AHEAD) row1 = row_at(nxt, tid);
    }
    f32x4_t acc[IN][IM] = {};
    for (int b = cur.b0; b < cur.b1; ++b, buf = buf + 1 < S ? buf + 1 : 0) {
      if (AHEAD && b + 1 == cur.b1) rows[tid] = row1;
      // This step's tiles have landed (all but the S - 2 steps of loads behind them; with two buffers a tile's first
      // step landed before the stores of the tile before, whose end it does not wait for), and every wave is done
      // reading the buffer that the next loads overwrite.
      if constexpr (S > 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((S - 2) * LW) : "memory");
      else if (b > cur.b0) asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      else asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const float* sx = (const float*)(f8_lds + buf * BYTES + (BN + BM) * 128) + wm * TM + c;
      float f[IM][2];
#pragma unroll
      for (int j = 0; j < IM; ++j) {
        f[j][0] = sx[j * 16] * wc[0];
        if constexpr (MODE == 1) f[j][1] = sx[j * 16] * wc[1];
      }
      // what is loaded now: S - 1 steps on; past the end the next tile's first step, or the last step again, read by
      // nobody (the count of loads in flight stays what the wait above takes it for)
      int bn = b + S - 1;
      if (bn >= cur.b1) {
        bn = more ? nxt.b0 : cur.b1 - 1;
        if (more) aim(nxt, true);
      }
      const int lbuf = buf > 0 ? buf - 1 : S - 1;
      scales(bn, lbuf);
      wscales(S == 2 ? bn : b + 1 < cur.b1 ? b + 1 : b);
      const uint8_t* ta = f8_lds + buf * BYTES;
      const uint8_t* tb = ta + BN * 128;
      auto arow = [&](int i) {
        return MODE == 1 ? (i < IN / 2 ? 0 : BN / 2) + wn * (TN / 2) + (i % (IN / 2)) * 16 + c : wn * TN + i * 16 + c;
      };
      i32x8_t fb[IM], fa[2];
      F8Wide wa, wb[WIDE ? IM : 1];
      f32x4_t p[2][IM];
#pragma unroll
      for (int j = 0; j < IM; ++j) {
        fb[j] = f8_frag(tb, wm * TM + j * 16 + c, g);
        if constexpr (WIDE) wb[j] = f8_widen(fb[j]);
      }
      fa[0] = f8_frag(ta, arow(0), g);
      auto fold = [&](int i, int j) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(p[i & 1][j][r], f[j][MODE == 1 && i >= IN / 2 ? 1 : 0], acc[i][j][r]);
      };
#pragma unroll
      for (int i = 0; i < IN; ++i) {
        // the next step's loads go out between the products: issued together they would fill the memory queue, and
        // no wave could start its products before most of them had been served; in the step's first half, so that the
        // last ones land in time (2048 x 14336 -> 4096 in 256 x 256 tiles 185 us, spread over the whole step 190)
#pragma unroll
        for (int l = spread(i); l < spread(i + 1); ++l) load(bn, lbuf, l);
        if (i + 1 < IN) fa[(i + 1) & 1] = f8_frag(ta, arow(i + 1), g);
        if constexpr (WIDE) wa = f8_widen(fa[i & 1]);
#pragma unroll
        for (int j = 0; j < IM; ++j) {
          if constexpr (WIDE) p[i & 1][j] = mfma_f8_wide(wa, wb[j], f32x4_t{});
          else p[i & 1][j] = mfma_f8_16x16x128(fa[i & 1], fb[j], f32x4_t{});
          if (i > 0) fold(i - 1, j);
        }
        // a row of products at a time (256 x 256), two for the smaller tiles (512 x 4096 -> 4096 in 128 x 128 32.5 -> 29.9 us)
        if (W == 8 || i & 1) __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < IM; ++j) fold(IN - 1, j);
    }
    // the buffer of the last step is the epilogue's, the other one holds the next tile's first step
    if constexpr (S > 2) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    f8_epilogue<BN, BM, WN, WM, MODE>(a, cur.m0, cur.mend, cur.n0, cur.split, f8_lds + (S == 2 ? buf ^ 1 : 0) * BYTES, acc);
    if (!more) return;
    cur = nxt;
  }
}

// LDS bytes of a workgroup.
constexpr int f8_tile_lds(int BN, int BM, int W, int S, int MODE) {
  return S * f8_stage_bytes(BN, BM) + (MODE == 1 && W == 8 ? 64 * W * 4 : 0);
}

// Workgroups for `tiles` tiles, in whole rounds of the XCDs: one a tile, or as many as run at once (by LDS and two waves a
// SIMD) where a workgroup takes tile after tile.
inline int64_t f8_tile_grid(int64_t tiles, int waves, int S, int lds, int cus) {
  if (S > 2) return imq_cdiv(tiles, 8) * 8;
  const int64_t a = 163840 / lds, b = 8 / waves, most = (int64_t)cus * (a < b ? a : b);
  return imq_cdiv(tiles < most ? tiles : most, 8) * 8;
}

}  // namespace
