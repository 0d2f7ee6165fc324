// Products with 8-bit operands for gfx950 (MI355X): the linear layer y = x W^T + b (+ GELU) from 8-bit tokens and
// weights, and its weight gradient dW = dY^T X from bf16 gradients and the 8-bit tokens that the layer read.
#include <algorithm>

#include "blocks8.hpp"

namespace fvsr {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
typedef __attribute__((address_space(3))) char lds_char;

// s_waitcnt lgkmcnt(0) vmcnt(0), then the workgroup barrier; memory accesses are not moved across it
__device__ __forceinline__ void wait_all_and_sync() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

__device__ __forceinline__ u32x4 make_rsrc(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)base;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)(const lds_char*)p);
}
// x, not known to be what it was before: what is computed from it in a loop is computed there, and takes no registers
// across it
__device__ __forceinline__ uint32_t afresh(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }
// 16 (or 4) bytes a lane from a buffer straight into LDS at `lds` + 16 (4) * lane; the address is the lane's offset
// plus the common one. The copy is waited for with vmcnt. One wait state has to pass between the write of M0 and its
// use, hence the s_nop.
__device__ __forceinline__ void copy16(u32x4 rsrc, uint32_t lds, uint32_t off, uint32_t common) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(uniform(lds)), "v"(off),
               "s"(rsrc), "s"(uniform(common)));
}
__device__ __forceinline__ void copy4(u32x4 rsrc, uint32_t lds, uint32_t off, uint32_t common) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds" ::"s"(uniform(lds)), "v"(off),
               "s"(rsrc), "s"(uniform(common)));
}

struct Linear8Args {
  In8 x, w;
  int64_t rows;
  int N, runs, ss;       // output features; runs and scale bytes a row of both operands
  const void* bias;      // may be null
  int bias_f32, gelu;
  void* y;
  int tiles_m, tiles_n;
  int part_runs;         // runs of a part, whole words of scales (linear8_kernel; part p writes its own rows x N sums at y)
};

// 0.5 y (1 + tanh(sqrt(2 / pi) (y + 0.044715 y^3))) = y / (1 + exp(-2 sqrt(2 / pi) (y + 0.044715 y^3))), the
// exponential in base 2: its argument overflows to +inf (the result then is 0) only where y is far below zero
__device__ __forceinline__ float gelu_tanh(float y) {
  constexpr float k = -2.f * 0.7978845608028654f * 1.4426950408889634f;
  const float e = __builtin_amdgcn_exp2f(k * y * fmaf(0.044715f * y, y, 1.f));
  return y * __builtin_amdgcn_rcpf(1.f + e);
}

// of 8 values, the steps side by side: an exponential or a reciprocal is used three instructions after it was asked for
// at the least
__device__ __forceinline__ void gelu_tanh8(float (&y)[8]) {
  constexpr float k = -2.f * 0.7978845608028654f * 1.4426950408889634f;
  float e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k * y[i] * fmaf(0.044715f * y[i], y[i], 1.f);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_exp2f(e[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = __builtin_amdgcn_rcpf(1.f + e[i]);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] *= e[i];
}

// bias (fp32, in LDS, at this lane's first feature), GELU and the store of a wave's fragments: this lane's features n0
// + 32 p .. + 7 (two fragments) of the tokens row0 + 16 m. WHOLE: every feature and token is inside.
template <bool GELU, bool WHOLE, int FN, int FM, typename O>
__device__ __forceinline__ void write_fragments(const Linear8Args& a, const f32x4 (&acc)[FN][FM], O* y, const float* bias, int n0,
                                                int64_t row0) {
  float b[FN / 2][8];
#pragma unroll
  for (int p = 0; p < FN / 2; ++p) {
    *(f32x4*)b[p] = *(const f32x4*)(bias + 32 * p);
    *(f32x4*)(b[p] + 4) = *(const f32x4*)(bias + 32 * p + 4);
  }
  O* out0 = y + row0 * a.N + n0;
  const int64_t step = (int64_t)16 * a.N;
#pragma unroll
  for (int m = 0; m < FM; ++m, out0 += step) {
    if (!WHOLE && row0 + 16 * m >= a.rows) continue;
#pragma unroll
    for (int p = 0; p < FN / 2; ++p) {
      float s[8];
      O v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] = acc[2 * p + (e >> 2)][m][e & 3] + b[p][e];
      if constexpr (GELU) gelu_tanh8(s);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (O)s[e];
      O* const out = out0 + 32 * p;
      const int n = n0 + 32 * p;
      if (WHOLE || n + 8 <= a.N) {
        *(any16*)out = *(u32x4*)v;
        if constexpr (sizeof(O) == 4) ((any16*)out)[1] = ((u32x4*)v)[1];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < a.N) out[e] = v[e];
      }
    }
  }
}
// true: by whole vectors (FN / 2 * FM * sizeof(O) / 2 stores)
template <bool GELU, int FN, int FM, typename O>
__device__ __forceinline__ bool write_tile(const Linear8Args& a, const f32x4 (&acc)[FN][FM], O* y, const float* bias, int n0,
                                           int64_t row0, bool whole) {
  if (whole) write_fragments<GELU, true>(a, acc, y, bias, n0, row0);
  else write_fragments<GELU, false>(a, acc, y, bias, n0, row0);
  return whole;
}

// Tile of TN output features x TM tokens, WN x WM waves; a step is one run: 128 codes of every row, and their scales in
// the matrix instruction.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 D (16 x 16) += A (16 x 128) B (128 x 16): lane l gives 32 codes of row l % 16 of A
// and of column l % 16 of B, and the scale byte of its 32 codes, taken from byte OP of a register; all of a run have
// one scale, so which 32 codes go with which lane does not matter as long as A and B agree. A is the weights: a lane's
// 4 results are then 4 features of one token. Fragment f of a wave holds the features 32 (f / 2) + 8 (i / 4) + 4 (f %
// 2) + i % 4, i = 0 .. 15, so that two fragments leave a lane 8 adjacent features: 16-byte stores, 64 bytes a token and
// instruction.
//
// LDS holds two steps: rows of 128 bytes, the 16-byte chunks XOR-ed by a number of the row under which the 16 rows that
// one instruction reads fall on 16 places of the 64 banks; copies go from memory to LDS directly (the XOR is on the
// source side), the next step's while this one's products run. A word of scales holds 4 steps.
//
// Sums are fp32. Before it adds them, the matrix core cuts each of the 8 products of an octet (8 adjacent codes of a
// lane) toward zero to a multiple of 2^(E - 13), E the largest sum of two code exponents among them (found by comparing
// 102400 random octets bit by bit; the 32 x 32 x 64 form and the unscaled ones do the same), so an octet is off by less
// than 2^-10 of its largest product. The rate of these instructions is why the layer is kept in 8 bits at all. Of a
// layer of random operands the fp32 sums are off by 5e-5 to 8e-5 (root mean square, relative), which an fp32 y carries
// and which moves 1 in 40 values of a bf16 y to the next number.
//
// Bound by latency where there is little work: 512 x 4096 x 1536, 12.3 us in 4 parts of 8 steps, 0.5 PFLOP/s.
template <int TN, int TM, int WN, int WM, bool GELU, typename O>
__global__ __launch_bounds__(64 * WN * WM, 2) void linear8_kernel(Linear8Args a) {
  constexpr int kWaves = WN * WM, FN = TN / WN / 16, FM = TM / WM / 16;
  static_assert(FN % 2 == 0 && TN % (8 * kWaves) == 0 && TM % (8 * kWaves) == 0, "tile");
  static_assert((TN + TM) / kWaves <= 64 && TN % ((TN + TM) / kWaves) == 0, "a wave's rows of scales belong to one operand");
  constexpr int kStage = (TN + TM) * kRun, kScales = (TN + TM) * 4;
  __shared__ __align__(1024) char sm[2 * kStage + 2 * kScales + TN * 4];
  float* const bias = (float*)(sm + 2 * kStage + 2 * kScales);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // tiles: every XCD a contiguous range, ordered in bands of 8 tiles of tokens so that a band's codes and the weights
  // stay in its L2
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  constexpr int kBand = 8;
  const int band = t / (kBand * a.tiles_n), in_band = t % (kBand * a.tiles_n);
  const int band_m = min(kBand, a.tiles_m - band * kBand);
  const int tm = band * kBand + in_band % band_m, tn = in_band / band_m;
  const int64_t m0 = (int64_t)tm * TM;
  const int n0 = tn * TN;
  const int ld = a.runs * kRun;
  const int rows_m = (int)min((int64_t)TM, a.rows - m0), rows_n = min(TN, a.N - n0);
  const u32x4 rw = make_rsrc(a.w.codes + (int64_t)n0 * ld, (uint32_t)rows_n * ld);
  const u32x4 rx = make_rsrc(a.x.codes + m0 * ld, (uint32_t)rows_m * ld);
  const u32x4 sw = make_rsrc(a.w.scales + (int64_t)n0 * a.ss, (uint32_t)rows_n * a.ss);
  const u32x4 sx = make_rsrc(a.x.scales + m0 * a.ss, (uint32_t)rows_m * a.ss);
  const uint32_t lds0 = lds_offset(sm);

  auto swz = [](int i, int q) { return ((i >> 1) & 1) | ((q >> 1) << 1) | (((q ^ (q >> 1)) & 1) << 2); };
  auto swz_w = [&](int r) { return swz(r & 3, (r >> 3) & 3); };
  auto swz_x = [&](int r) { return swz(r & 3, (r >> 2) & 3); };
  // a lane's source offsets: of 8 rows a wave and copy, and of a word of scales a row. Rows past the last one read it
  // again (their results are not stored).
  constexpr int kCW = TN / (8 * kWaves), kCX = TM / (8 * kWaves), kScaleRows = (TN + TM) / kWaves;
  uint32_t ow[kCW], ox[kCX];
#pragma unroll
  for (int c = 0; c < kCW; ++c) {
    const int r = (c * kWaves + wave) * 8 + (lane >> 3);
    ow[c] = (uint32_t)(min(r, rows_n - 1) * ld + (((lane & 7) ^ swz_w(r)) << 4));
  }
#pragma unroll
  for (int c = 0; c < kCX; ++c) {
    const int r = (c * kWaves + wave) * 8 + (lane >> 3);
    ox[c] = (uint32_t)(min(r, rows_m - 1) * ld + (((lane & 7) ^ swz_x(r)) << 4));
  }
  const int sr = wave * kScaleRows + (lane & (kScaleRows - 1));   // this lane's row of scales
  const bool s_of_w = wave * kScaleRows < TN;
  const uint32_t so = (uint32_t)((s_of_w ? min(sr, rows_n - 1) : min(sr - TN, rows_m - 1)) * a.ss);
  const u32x4 rs = s_of_w ? sw : sx;
  auto copy_step = [&](int k) {
    const uint32_t base = lds0 + (k & 1) * kStage + wave * 8 * kRun;
    static_for<0, kCW>([&](auto c) { copy16(rw, base + c * kWaves * 8 * kRun, ow[c], k * kRun); });
    static_for<0, kCX>([&](auto c) { copy16(rx, base + TN * kRun + c * kWaves * 8 * kRun, ox[c], k * kRun); });
    if ((k & 3) == 0 && lane < kScaleRows)
      copy4(rs, lds0 + 2 * kStage + ((k >> 2) & 1) * kScales + wave * kScaleRows * 4, so, k);
  };

  const int wn = wave % WN, wm = wave / WN, i = lane & 15, g = lane >> 4;
  const int rw0 = wn * (TN / WN) + ((i >> 2) << 3) + (i & 3), rx0 = wm * (TM / WM) + i;
  const char* pw[2];
  const char* px[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pw[h] = sm + rw0 * kRun + (((2 * g + h) ^ swz_w(rw0)) << 4);
    px[h] = sm + TN * kRun + rx0 * kRun + (((2 * g + h) ^ swz_x(rx0)) << 4);
  }
  f32x4 acc[FN][FM];
#pragma unroll
  for (int f = 0; f < FN; ++f)
#pragma unroll
    for (int m = 0; m < FM; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};

  const int k_from = blockIdx.y * a.part_runs, k_to = min(a.runs, k_from + a.part_runs);
  copy_step(k_from);
  for (int n = threadIdx.x; n < TN; n += 64 * kWaves)
    bias[n] = !a.bias || n0 + n >= a.N ? 0.f : a.bias_f32 ? ((const float*)a.bias)[n0 + n] : (float)((const bf16*)a.bias)[n0 + n];
  int qw[FN], qx[FM];
  for (int k0 = k_from; k0 < k_to; k0 += 4) {
    static_for<0, 4>([&](auto kc) {
      constexpr int OP = decltype(kc)::value;
      const int k = k0 + OP;
      if (k >= k_to) return;
      wait_all_and_sync();   // step k is in LDS, and nobody reads step k - 1 any more
      if (k + 1 < k_to) copy_step(k + 1);
      if constexpr (OP == 0) {
        const char* ps = sm + 2 * kStage + ((k >> 2) & 1) * kScales;
#pragma unroll
        for (int f = 0; f < FN; ++f) qw[f] = *(const int*)(ps + 4 * (rw0 + (f >> 1) * 32 + (f & 1) * 4));
#pragma unroll
        for (int m = 0; m < FM; ++m) qx[m] = *(const int*)(ps + 4 * (TN + rx0 + 16 * m));
      }
      const int st = (k & 1) * kStage;
      auto read = [&](const char* const (&p)[2], int off) {
        const u32x4 lo = *(const u32x4*)(p[0] + off), hi = *(const u32x4*)(p[1] + off);
        return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
      };
      i32x8 fw[FN];
#pragma unroll
      for (int f = 0; f < FN; ++f) fw[f] = read(pw, st + ((f >> 1) * 32 + (f & 1) * 4) * kRun);
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        const i32x8 fx = read(px, st + 16 * m * kRun);
#pragma unroll
        for (int f = 0; f < FN; ++f)
          acc[f][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[f], fx, acc[f][m], 0, 0, OP, qw[f], OP, qx[m]);
      }
    });
  }

  const int fn = wn * (TN / WN) + 8 * g;
  write_tile<GELU>(a, acc, (O*)a.y + blockIdx.y * a.rows * a.N, bias + fn, n0 + fn, m0 + rx0,
                   rows_m == TM && rows_n == TN);
}

// The large product: 256 features x 256 tokens a tile, one workgroup a CU walking over tiles without a break between
// them. Two groups of four waves, one of each on every SIMD, take turns: while one group's 32 matrix instructions of a
// step (a run: 128 codes of every row) go, the other reads its operands of the step into registers and asks for later
// ones. A phase ends with a barrier; steps s are counted across tiles, LDS holds two of them, and wave w of a group
// computes features 64 w .. 64 w + 63 of the group's 128 tokens:
//
//   phase      2s                                       2s + 1
//   group 0    copy group 1's tokens of s + 1, read(s)  multiply(s)
//   group 1    multiply(s - 1)                          copy group 0's tokens of s + 2, read(s), copy the weights of s + 2
//
// Everything is asked for as soon as its place is free: group 0's tokens of step s have been read when phase 2s ends,
// group 1's when phase 2s + 1 ends; the weights that wave w of group 1 reads in phase 2s + 1 wave w of group 0 has read
// before, so it replaces them at once. Each is needed about three phases later, and its wave waits for it at the end of
// that time, by the count of what it has asked for since (memory operations of a wave complete in order). A group
// writes its tile, and starts the next one, in its read phase, under the other group's products.
//
// 8192^3 in 382-394 us by part (2.8-2.9 PFLOP/s), 17280 x 8960 x 1536 in 207-210 (2.3, 408 tiles: a round and 152
// over), 17280 x 1536 x 8960 in 228 (2.1, 12 steps a tile) and with GELU 237-247, the matrix cores busy 44 % of the
// cycles in the last; no bank conflicts. What bounds the first, 64 steps a tile, is the issue of the copies and the
// reads from LDS side by side: where it took 382, without the copies of one operand (of both) 330 (303) us, without any
// wait for them 372. At 12 steps a tile this was not told apart.
template <bool GELU, typename O>
__global__ __launch_bounds__(512, 2) void linear8_large_kernel(Linear8Args a) {
  constexpr int FN = 4, FM = 8, kStores = FN / 2 * FM * (int)sizeof(O) / 2;
  constexpr int kBuf = 256 * kRun;                         // one operand's rows of a step
  constexpr int kX = 2 * kBuf, kS = 4 * kBuf;              // LDS: weights of two steps, tokens of two steps,
  constexpr int kScales = 512 * 4, kB = kS + 4 * kScales;  // scales of 4 x 4 steps, biases of 4 tiles
  __shared__ __align__(1024) char sm[kB + 4 * 1024];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave >> 2, w = wave & 3, i = lane & 15, g = lane >> 4;
  const int G = a.runs, ld = G * kRun;
  const uint32_t lds0 = lds_offset(sm);
  // chunk c of row r of the weights lies at c ^ swz(r % 4, r / 8 % 4), of the tokens at c ^ swz(r % 4, r / 4 % 4): the
  // 16 rows that a cycle of a 16-byte read serves (of a fragment: features 8 (i / 4) + i % 4, tokens i) then lie on
  // different banks
  auto swz = [](int r, int q) { return ((r >> 1) & 1) | ((q >> 1) << 1) | (((q ^ (q >> 1)) & 1) << 2); };
  const int rw0 = w * 64 + ((i >> 2) << 3) + (i & 3), rx0 = group * 128 + i;
  const char* pw[2];
  const char* px[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pw[h] = sm + rw0 * kRun + (((2 * g + h) ^ swz(rw0 & 3, (rw0 >> 3) & 3)) << 4);
    px[h] = sm + kX + rx0 * kRun + (((2 * g + h) ^ swz(rx0 & 3, (rx0 >> 2) & 3)) << 4);
  }
  // copies: 8 rows an instruction, this wave's 64 rows of weights and 32 of the other group's tokens; a lane's source
  // of rows 8 c + r8 is 8 c rows on, its chunk XOR-ed by what c adds to swz
  const int r8 = lane >> 3, cs = ((lane & 7) ^ ((r8 >> 1) & 1)) << 4;
  const uint32_t ow = (uint32_t)(r8 * ld + cs), ox = (uint32_t)(r8 * ld + (cs ^ ((r8 >> 2) << 6)));
  const uint32_t os = (uint32_t)(lane * a.ss);

  // this workgroup's tiles: every XCD walks over a contiguous range of them, in bands of 8 tiles of tokens
  const int tiles = a.tiles_m * a.tiles_n;
  const int xcd = blockIdx.x % kXcds, per = (int)gridDim.x / kXcds;   // the grid is a multiple of the XCDs
  const int first = xcd * (tiles / kXcds) + min(xcd, tiles % kXcds);
  const int end = first + tiles / kXcds + (xcd < tiles % kXcds ? 1 : 0);
  int t = first + (int)blockIdx.x / kXcds;
  if (t >= end) return;   // the whole workgroup
  auto place = [&](int tile, int64_t& m0, int& n0) __attribute__((always_inline)) {
    constexpr int kBand = 8;
    const int band = tile / (kBand * a.tiles_n), in_band = tile % (kBand * a.tiles_n);
    const int band_m = min(kBand, a.tiles_m - band * kBand);
    m0 = (int64_t)(band * kBand + in_band % band_m) * 256;
    n0 = in_band / band_m * 256;
  };

  // what this wave asks for: step ck of tile ct; rows past the last one lie past the end of a buffer and are read as
  // zeros
  int ct = t, ck = 0, cn = 0, cs4 = 0;   // cn: tiles, cs4: words of scales asked for before
  int64_t cm0;
  int cn0;
  u32x4 dw, dx, dsw, dsx, db;
  auto source = [&]() __attribute__((always_inline)) {
    place(ct, cm0, cn0);
    auto rows = [&](int64_t have, int64_t at, int most) __attribute__((always_inline)) {
      return (uint32_t)max((int64_t)0, min(have - at, (int64_t)most));
    };
    const int64_t mx = cm0 + (1 - group) * 128 + w * 32;
    dx = make_rsrc(a.x.codes + mx * ld, rows(a.rows, mx, 32) * ld);
    if (group == 1) {
      const int nw = cn0 + w * 64;
      dw = make_rsrc(a.w.codes + (int64_t)nw * ld, rows(a.N, nw, 64) * ld);
      dsw = make_rsrc(a.w.scales + (int64_t)nw * a.ss, rows(a.N, nw, 64) * a.ss);
      dsx = make_rsrc(a.x.scales + (cm0 + w * 64) * a.ss, rows(a.rows, cm0 + w * 64, 64) * a.ss);
      db = make_rsrc(a.bias ? (const float*)a.bias + nw : nullptr, a.bias ? rows(a.N, nw, 64) * 4 : 0);
    }
  };
  auto advance = [&]() __attribute__((always_inline)) {
    if ((ck & 3) == 3 || ck + 1 == G) ++cs4;
    if (++ck < G) return;
    ck = 0;
    ++cn;
    ct += per;
    if (ct < end) source();
  };
  auto copy_tokens = [&](int par) __attribute__((always_inline)) {   // the other group's, 32 rows
    const uint32_t to = lds0 + kX + par * kBuf + ((1 - group) * 128 + w * 32) * kRun;
    const uint32_t o = afresh(ox);
    static_for<0, 4>([&](auto c) __attribute__((always_inline)) {
      copy16(dx, to + c * 8 * kRun, (o ^ ((c & 1) * 0x60)) + c * 8 * ld, ck * kRun);
    });
  };
  auto copy_small = [&]() __attribute__((always_inline)) {   // scales and biases (group 1), where a word or a tile begins
    if (ck & 3) return;
    const uint32_t to = lds0 + kS + (cs4 & 3) * kScales + w * 256;
    copy4(dsw, to, os, ck);
    copy4(dsx, to + 1024, os, ck);
    if (ck == 0) copy4(db, lds0 + kB + (cn & 3) * 1024 + w * 256, lane * 4, 0);
  };
  auto copy_weights = [&](int par) __attribute__((always_inline)) {
    const uint32_t to = lds0 + par * kBuf + w * 64 * kRun;
    const uint32_t o = afresh(ow);
    static_for<0, 8>([&](auto c) __attribute__((always_inline)) {
      constexpr int q = c & 3, m = (q >> 1) | (((q ^ (q >> 1)) & 1) << 1);
      copy16(dw, to + c * 8 * kRun, (o ^ (m << 5)) + c * 8 * ld, ck * kRun);
    });
  };

  i32x8 fw[FN], fx[FM];
  int qw[FN], qx[FM];
  f32x4 acc[FN][FM];
  int par = 0, rs4 = 0;
  auto read_step = [&](auto kc) __attribute__((always_inline)) {
    if constexpr (decltype(kc)::value == 0) {
      const char* s = sm + kS + (rs4 & 3) * kScales;
      ++rs4;
#pragma unroll
      for (int f = 0; f < FN; ++f) qw[f] = *(const int*)(s + 4 * (rw0 + (f >> 1) * 32 + (f & 1) * 4));
#pragma unroll
      for (int m = 0; m < FM; ++m) qx[m] = *(const int*)(s + 4 * (256 + rx0 + 16 * m));
    }
    const int st = par * kBuf;
    auto read = [&](const char* const (&p)[2], int off) {
      const u32x4 lo = *(const u32x4*)(p[0] + st + off), hi = *(const u32x4*)(p[1] + st + off);
      return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
#pragma unroll
    for (int f = 0; f < FN; ++f) fw[f] = read(pw, ((f >> 1) * 32 + (f & 1) * 4) * kRun);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < FM; ++m) fx[m] = read(px, 16 * m * kRun);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](auto kc, auto fresh) __attribute__((always_inline)) {
    constexpr int OP = decltype(kc)::value;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int m = 0; m < FM; ++m)
#pragma unroll
      for (int f = 0; f < FN; ++f) {
        const f32x4 c = decltype(fresh)::value ? f32x4{0.f, 0.f, 0.f, 0.f} : acc[f][m];
        acc[f][m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[f], fx[m], c, 0, 0, OP, qw[f], OP, qx[m]);
      }
    __builtin_amdgcn_s_setprio(0);
  };
  auto turn = [] {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#define FVSR_WAIT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")

  int64_t m0 = 0;
  int n0 = 0, bt = 0;   // the tile being computed, and how many before it
  bool held = false;    // its predecessor is still in acc
  // writes the tile in acc; whether it took exactly kStores stores
  auto write = [&]() __attribute__((always_inline)) {
    if (!held) return false;
    const float* b = (const float*)(sm + kB + ((bt - 1) & 3) * 1024);
    return write_tile<GELU>(a, acc, (O*)a.y, b + w * 64 + 8 * g, n0 + w * 64 + 8 * g, m0 + rx0,
                            m0 + 256 <= a.rows && n0 + 256 <= a.N);
  };

  source();
  if (group == 0) {
    copy_tokens(0);
    advance();
  } else {
    for (int s = 0; s < 2 && ct < end; ++s) {
      copy_small();
      copy_tokens(s);
      copy_weights(s);
      advance();
    }
  }
  FVSR_WAIT(0);
  turn();
  if (group == 1) turn();   // phase 0
  for (; t < end; t += per) {
    for (int k0 = 0; k0 < G; k0 += 4)
      static_for<0, 4>([&](auto kc) __attribute__((always_inline)) {
        const int k = k0 + kc;
        if (k >= G) return;
        const bool ask = ct < end;
        bool wrote = false;
        if constexpr (decltype(kc)::value == 0)
          if (k == 0) {
            wrote = write();
            place(t, m0, n0);
            held = true;
            ++bt;
          }
        read_step(kc);
        // then what has been asked for since the copies that the next phase needs may be outstanding: this step's, and
        // maybe stores
        if (group == 0) {
          if (ask) copy_tokens(par ^ 1);
          if (!ask) FVSR_WAIT(0);
          else if (wrote) FVSR_WAIT(4 + kStores);
          else FVSR_WAIT(4);
        } else {
          if (ask) {
            copy_small();
            copy_tokens(par);
            // the weights were read first: with 15 of the 24 reads outstanding, their place is free
            asm volatile("s_waitcnt lgkmcnt(15)" ::: "memory");
            copy_weights(par);
          }
          if (!ask) FVSR_WAIT(0);
          else if (wrote) FVSR_WAIT(12 + kStores);
          else FVSR_WAIT(12);
        }
        if (ask) advance();
        turn();
        if constexpr (decltype(kc)::value == 0) {
          if (k == 0) multiply(kc, std::true_type{});
          else multiply(kc, std::false_type{});
        } else {
          multiply(kc, std::false_type{});
        }
        par ^= 1;
        if (group == 0 || k + 1 < G || t + per < end) turn();
      });
  }
  write();
#undef FVSR_WAIT
}

__global__ __launch_bounds__(256) void widen_kernel(const bf16* __restrict__ in, int n, float* __restrict__ out) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < n) out[i] = (float)in[i];
}

// y = the sum over parts of their (rows, N) sums, bias, GELU; V elements a thread (4 where N is a multiple of 4)
template <int V, typename O>
__global__ __launch_bounds__(256) void linear8_join_kernel(const float* __restrict__ part, int parts, int64_t n, int N,
                                                           const void* __restrict__ bias, int bias_f32, int gelu,
                                                           O* __restrict__ y) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= n) return;
  typedef float fv __attribute__((ext_vector_type(V)));
  fv s = *(const fv*)(part + i);
  for (int p = 1; p < parts; ++p) s += *(const fv*)(part + p * n + i);
  const int c = (int)(i % N);
#pragma unroll
  for (int e = 0; e < V; ++e) {
    float t = s[e];
    if (bias) t += bias_f32 ? ((const float*)bias)[c + e] : (float)((const bf16*)bias)[c + e];
    if (gelu) t = gelu_tanh(t);
    y[i + e] = (O)t;
  }
}

// The product of a few tokens (16 * FM at most), bound by reading the weights: 16 features a workgroup, its four waves
// take every fourth run and read their operands straight into registers, up to three runs asked for at once; the waves'
// sums meet in LDS. 1 x 1536 x 9216: 5.8 us, 2.5 TB/s (a chain of three round trips; in tiles of 128 x 128 9.9 us).
template <int FM, typename O>
__global__ __launch_bounds__(256) void linear8_few_kernel(Linear8Args a) {
  __shared__ float sm[4][FM][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, ld = a.runs * kRun;
  const int rows = (int)a.rows;
  // rows past the last one read it again: their results are not stored
  const int n = min(n0 + i, a.N - 1);
  const uint8_t* const w = a.w.codes + (int64_t)n * ld + g * 32;
  const uint8_t* const ws = a.w.scales + (int64_t)n * a.ss;
  f32x4 acc[FM];
#pragma unroll
  for (int m = 0; m < FM; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
  constexpr int U = FM < 4 ? 3 : 2;   // runs asked for at once
  for (int k0 = wave; k0 < a.runs; k0 += 4 * U) {
    i32x8 fw[U], fx[U][FM];
    int qw[U], qx[U][FM];
    auto load = [](const uint8_t* p) {
      const u32x4 lo = *(const u32x4*)p, hi = *(const u32x4*)(p + 16);
      return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
    };
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = min(k0 + 4 * u, a.runs - 1);   // past the last one: asked for again, and not used
      fw[u] = load(w + k * kRun);
      qw[u] = ws[k];
#pragma unroll
      for (int m = 0; m < FM; ++m) {
        const int64_t row = min(16 * m + i, rows - 1);
        fx[u][m] = load(a.x.codes + row * ld + g * 32 + k * kRun);
        qx[u][m] = a.x.scales[row * a.ss + k];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k0 + 4 * u < a.runs)
#pragma unroll
        for (int m = 0; m < FM; ++m)
          acc[m] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fw[u], fx[u][m], acc[m], 0, 0, 0, qw[u], 0, qx[u][m]);
  }
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int e = 0; e < 4; ++e) sm[wave][m][i][4 * g + e] = acc[m][e];   // token i, feature 4 g + e
  __syncthreads();
#pragma unroll
  for (int m = 0; m < FM; ++m) {
    const int token = threadIdx.x >> 4, f = threadIdx.x & 15, row = 16 * m + token;
    if (row >= rows || n0 + f >= a.N) continue;
    float s = (sm[0][m][token][f] + sm[1][m][token][f]) + (sm[2][m][token][f] + sm[3][m][token][f]);
    if (a.bias) s += a.bias_f32 ? ((const float*)a.bias)[n0 + f] : (float)((const bf16*)a.bias)[n0 + f];
    if (a.gelu) s = gelu_tanh(s);
    ((O*)a.y)[(int64_t)row * a.N + n0 + f] = (O)s;
  }
}

// How a product is cut up. A few tokens: by 16 features. Else tiles of 256 x 256, one a CU, or of 128 x 128, two a CU:
// a round of the former does twice the work of one of the latter in 1.5 to 1.6 times its time (8192^3, 4 rounds against
// 8: 382 us, 518; 4096 x 1536 x 6144, 2 against 3: 48 us, 46), so by the rounds that each needs. Where there are few of
// the latter, each row's runs are cut into parts of at least 8 (512 x 4096 x 1536, 48 tiles: 12.3 us in 4 parts and 4.2
// to join them, 25 in one).
struct Linear8Plan {
  bool few, large;
  int64_t tiles;
  int parts, part_runs;
};
static Linear8Plan linear8_plan(int64_t rows, int K, int N) {
  auto tiles_of = [&](int t) { return ceil_div(rows, t) * ceil_div(N, t); };
  Linear8Plan p{};
  p.few = rows <= 64;
  p.large = ceil_div(tiles_of(256), 256) * 8 <= ceil_div(tiles_of(128), 512) * 5;
  p.tiles = tiles_of(p.large ? 256 : 128);
  const int runs = runs_of(K);
  int64_t parts = 1;
  if (!p.few && !p.large && p.tiles < 256) parts = std::max<int64_t>(1, std::min<int64_t>(256 / p.tiles, runs / 8));
  p.part_runs = (int)ceil_div(ceil_div(runs, 4), parts) * 4;
  p.parts = (int)ceil_div(runs, p.part_runs);
  return p;
}

size_t linear8_workspace(int64_t rows, int K, int N) {
  const Linear8Plan p = linear8_plan(rows, K, N);
  if (p.few) return 0;
  return p.large ? (size_t)N * sizeof(float) : p.parts > 1 ? (size_t)p.parts * rows * N * sizeof(float) : 0;
}

int launch_linear8(In8 x, int64_t rows, int K, In8 w, int N, int bias_dtype, const void* bias, int gelu, int out_dtype,
                   void* y, void* ws, hipStream_t stream) {
  if (rows <= 0) return FVSR_OK;
  const Linear8Plan p = linear8_plan(rows, K, N);
  Linear8Args a{};
  a.x = x; a.w = w; a.rows = rows; a.N = N; a.runs = runs_of(K); a.ss = scale_stride(K);
  a.bias = bias; a.bias_f32 = bias_dtype == FVSR_DTYPE_F32; a.gelu = gelu; a.y = y;
  a.part_runs = p.part_runs;
  if (!p.few && p.tiles >= 1 << 24) return set_error(FVSR_ERR_UNSUPPORTED, "linear8: too many output tiles for one launch");
  const bool bf = out_dtype == FVSR_DTYPE_BF16;
  const int T = p.large ? 256 : 128;
  a.tiles_m = (int)ceil_div(rows, T);
  a.tiles_n = (int)ceil_div(N, T);
  if (p.few) {
    const dim3 grid((unsigned)ceil_div(N, 16));
    auto go = [&](auto fm) {
      constexpr int FM = decltype(fm)::value;
      if (bf) hipLaunchKernelGGL((linear8_few_kernel<FM, bf16>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((linear8_few_kernel<FM, float>), grid, dim3(256), 0, stream, a);
    };
    if (rows <= 16) go(std::integral_constant<int, 1>{});
    else if (rows <= 32) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 4>{});
  } else if (p.large) {
    if (bias && !a.bias_f32) {
      hipLaunchKernelGGL(widen_kernel, dim3((unsigned)ceil_div(N, 256)), dim3(256), 0, stream, (const bf16*)bias, N, (float*)ws);
      a.bias = ws;
    }
    const dim3 grid((unsigned)std::min<int64_t>(256, ceil_div(p.tiles, kXcds) * kXcds));
    auto go = [&](auto g) {
      constexpr bool G = decltype(g)::value;
      if (bf) hipLaunchKernelGGL((linear8_large_kernel<G, bf16>), grid, dim3(512), 0, stream, a);
      else hipLaunchKernelGGL((linear8_large_kernel<G, float>), grid, dim3(512), 0, stream, a);
    };
    if (gelu) go(std::true_type{});
    else go(std::false_type{});
  } else if (p.parts > 1) {
    Linear8Args part = a;
    part.bias = nullptr;
    part.gelu = 0;
    part.y = ws;
    hipLaunchKernelGGL((linear8_kernel<128, 128, 4, 2, false, float>), dim3((unsigned)p.tiles, (unsigned)p.parts), dim3(512),
                       0, stream, part);
    FVSR_HIP_CHECK(hipGetLastError());
    const int64_t n = rows * N;
    auto join = [&](auto v, auto o) {
      constexpr int V = decltype(v)::value;
      using O = decltype(o);
      hipLaunchKernelGGL((linear8_join_kernel<V, O>), dim3((unsigned)ceil_div(n, 256 * V)), dim3(256), 0, stream, (const float*)ws,
                         p.parts, n, N, bias, a.bias_f32, gelu, (O*)y);
    };
    auto with = [&](auto o) {
      if (N % 4 == 0) join(std::integral_constant<int, 4>{}, o);
      else join(std::integral_constant<int, 1>{}, o);
    };
    if (bf) with(bf16{});
    else with(float{});
  } else {
    // where a CU has one workgroup at most, 8 waves of it: two on each SIMD, whose reads and products overlap (512 x
    // 1536 x 1536, 12 steps: 9.8 us with 8 waves, 10.5 with 4)
    const dim3 grid((unsigned)p.tiles);
    auto go = [&](auto wn, auto g) {
      constexpr int WN = decltype(wn)::value;
      constexpr bool G = decltype(g)::value;
      if (bf) hipLaunchKernelGGL((linear8_kernel<128, 128, WN, 2, G, bf16>), grid, dim3(128 * WN), 0, stream, a);
      else hipLaunchKernelGGL((linear8_kernel<128, 128, WN, 2, G, float>), grid, dim3(128 * WN), 0, stream, a);
    };
    auto with = [&](auto wn) { gelu ? go(wn, std::true_type{}) : go(wn, std::false_type{}); };
    if (p.tiles <= 256) with(std::integral_constant<int, 4>{});
    else with(std::integral_constant<int, 2>{});
  }
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

// ------------------------------------------------------------------------------------------------------------
// weight gradient
// ------------------------------------------------------------------------------------------------------------
struct WeightGradArgs {
  const bf16* dy;
  int ld;                    // elements from one of its rows to the next
  In8 x;
  int64_t rows, part_rows;   // part_rows: tokens of a part (the work is split over parts where there are few tiles), whole steps
  int N, K, runs, ss;
  void* dw;                  // (parts, N, K), fp32 where there are more than one
  float* db;                 // (parts * tiles_k, N) or null
  int tiles_n, tiles_k;
};

// the first `n` of 4 results, at any address
template <typename O>
__device__ __forceinline__ void store4(O* out, f32x4 x, int n) {
  O v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (O)x[e];
  if (n >= 4) {
    if constexpr (sizeof(O) == 4) *(any16*)out = *(u32x4*)v;
    else *(any8*)out = *(u32x2*)v;
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) out[e] = v[e];
  }
}

// dW (N, K) = dY^T X, 256 features x 256 channels a workgroup, steps of 64 tokens. Both operands lie token-major, so
// the product's depth runs across rows: they are kept in LDS as they come, [token][column], in bf16 (codes times scales
// are exact in it), and ds_read_b64_tr_b16 hands a lane 4 tokens of one column: 16 lanes read 4 rows of 16 columns,
// lane i gets column i of the four. Two groups of four waves take turns as in linear8_large_kernel; wave w of group h
// computes features 64 w .. 64 w + 63 and channels 128 h .. 128 h + 127, a run:
//
//   phase      2s                                                          2s + 1
//   group 0    widen X1(s), read(s), ask for dY(s + 1) and codes of s + 2  multiply(s)
//   group 1    multiply(s - 1)                                             widen X0(s + 1), read(s), ask for codes of s + 3
//
// LDS: dY of two steps, in blocks of 64 features (rows of 128 bytes, a token each). X as bf16, a half (a group's run)
// of one step each: written in the phases in which it is not read. Codes and scales as they come, two steps: a wave
// copies, and later widens, its own 16 tokens of the other group's half, so its own count of copies is all it waits
// for. The 32-byte pairs of a row of token t are XOR-ed by (t / 2 % 2, t / 8 % 2): a half wave's transposing read (4
// tokens of 16 columns for each 16 lanes) then touches every bank once. dY's copies stand between the reads from LDS:
// behind them, at the phase's end, their issue was what the other group waited for (497 us at 17280 x 1536 x 8960, now
// 434: 1.1 PFLOP/s on 210 of 256 CUs, which alone allows 1.3 of the 1.58 that a library product of 16384^3 reaches;
// matrix cores busy 53 % of those CUs' cycles).
// Copies past the last token read zeros (and nothing else), so every phase asks for the same number. db: a step's
// column sums are taken by one of the tiles_k workgroups that read the step, from the fragments in registers, under the
// products (a column a lane; as products with rows of ones and zeros an infinity would reach other columns).
template <typename O>
__global__ __launch_bounds__(512, 2) void weight_grad_kernel(WeightGradArgs a) {
  constexpr int FN = 4, FM = 8, kTokens = 64;
  constexpr int kBlk = kTokens * 128;                       // 64 columns (bf16) of a step
  constexpr int kX = 8 * kBlk;                              // LDS: dY 2 x 4 blocks, X 2 halves x 2 blocks,
  constexpr int kRaw = 12 * kBlk, kSc = kRaw + 2 * 2 * kBlk;   // codes 2 halves x 2 steps, scales 2 halves x 2 steps x 64 words
  __shared__ __align__(1024) char sm[kSc + 4 * 256];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave >> 2, w = wave & 3, i = lane & 15, g = lane >> 4;
  const uint32_t lds0 = lds_offset(sm);
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tk = t % a.tiles_k, tn = t / a.tiles_k, n0 = tn * 256 + w * 64, k0 = tk * 256;
  const int64_t from = (int64_t)blockIdx.y * a.part_rows, to = min(a.rows, from + a.part_rows);
  const int steps = (int)((to - from + kTokens - 1) / kTokens);
  const int ldn = a.ld * 2, ldk = a.runs * kRun;
  const int other = 1 - group;

  // copies: 8 tokens an instruction
  const int r8 = lane >> 3, c8 = lane & 7;
  const uint32_t od = (uint32_t)((((c8 >> 1) ^ ((r8 >> 1) & 1)) << 5) | ((c8 & 1) << 4));   // in a row of dY's block
  const uint32_t oc = (uint32_t)((16 * w + r8) * ldk + c8 * 16);
  const int run = tk * 2 + other;                           // this wave's codes' run
  const int count = (int)(to - from);                       // tokens (a part has fewer than 2^31)
  // dY, codes and scales of the step that is asked for next, and their places in LDS: steps are asked for in order, so
  // all that a step costs is three sums (its 64-bit products and minima each time cost 60 us of 445)
  auto records = [&](int left, int ld, int off) __attribute__((always_inline)) {
    return (uint32_t)max(0, max(0, min(kTokens, left)) * ld - off);
  };
  auto move = [](u32x4& d, int by) __attribute__((always_inline)) {
    const uint64_t b = (((uint64_t)d[1] << 32) | d[0]) + (uint64_t)by;
    d[0] = (uint32_t)b;
    d[1] = (uint32_t)(b >> 32);
  };
  int dy_left = count, codes_left = count;
  u32x4 dd = make_rsrc(a.dy + from * a.ld + n0, records(count, ldn, n0 * 2));
  u32x4 dc = make_rsrc(a.x.codes + from * ldk + run * kRun, records(count, ldk, run * kRun));
  u32x4 ds = make_rsrc(a.x.scales + from * a.ss + (run & ~3), records(count, a.ss, run & ~3));
  uint32_t dy_at = lds0 + w * kBlk, dy_flip = 4 * kBlk;
  uint32_t codes_at = lds0 + kRaw + other * kBlk + w * 2048, codes_flip = 2 * kBlk;
  uint32_t scales_at = lds0 + kSc + other * 256 + w * 64, scales_flip = 2 * 256;
  auto next_dy = [&]() __attribute__((always_inline)) {
    move(dd, kTokens * ldn);
    dy_left -= kTokens;
    if (dy_left < kTokens) dd[2] = records(dy_left, ldn, n0 * 2);
    dy_at += dy_flip;
    dy_flip = 0u - dy_flip;
  };
  auto next_codes = [&]() __attribute__((always_inline)) {
    move(dc, kTokens * ldk);
    move(ds, kTokens * a.ss);
    codes_left -= kTokens;
    if (codes_left < kTokens) {
      dc[2] = records(codes_left, ldk, run * kRun);
      ds[2] = records(codes_left, a.ss, run & ~3);
    }
    codes_at += codes_flip;
    codes_flip = 0u - codes_flip;
    scales_at += scales_flip;
    scales_flip = 0u - scales_flip;
  };
  auto copy_dy = [&](auto c) __attribute__((always_inline)) {   // 8 of its 64 tokens
    copy16(dd, dy_at + c * 1024, (afresh(od) ^ ((c & 1) << 6)) + (r8 + c * 8) * ldn, 0);
  };
  auto copy_codes = [&](auto c) __attribute__((always_inline)) {   // 0, 1: 8 tokens' codes; 2: this wave's 16 scales
    if constexpr (decltype(c)::value < 2) copy16(dc, codes_at + c * 1024, afresh(oc) + c * 8 * ldk, 0);
    else if (lane < 16) copy4(ds, scales_at, (16 * w + afresh(lane)) * a.ss, 0);
  };
  // codes of step s, this wave's tokens 16 w + 8 j + lane / 8, 16 channels a lane, to bf16
  u32x4 raw[2];
  uint32_t raw_scale[2];
  auto read_codes = [&](int s) __attribute__((always_inline)) {
    const int l = (int)afresh(threadIdx.x & 63);
    const char* r = sm + kRaw + ((s & 1) * 2 + other) * kBlk + w * 2048 + l * 16;
    const char* sc = sm + kSc + ((s & 1) * 2 + other) * 256 + w * 64 + (l >> 3) * 4 + (run & 3);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      raw[j] = *(const u32x4*)(r + j * 1024);
      raw_scale[j] = *(const uint8_t*)(sc + j * 32);
    }
  };
  auto widen = [&]() __attribute__((always_inline)) {
    const int l = (int)afresh(threadIdx.x & 63), r = l >> 3, c = l & 7;
    char* out = sm + kX + other * 2 * kBlk + (c >> 2) * kBlk + (16 * w + r) * 128;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float by = __uint_as_float(raw_scale[j] << 23);
      bf16x2 v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[j][e], by, false);
        v[2 * e + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[j][e], by, true);
      }
      // the lanes of one block write the lower halves of their pairs first, those of the other, on the same banks, the
      // upper ones
      char* o = out + j * 1024 + (((c & 3) ^ ((r >> 1) & 1) ^ (j << 1)) << 5);
      const bool up = c >> 2;
      const u32x4 lo = *(u32x4*)v, hi = *(u32x4*)(v + 4);
      *(u32x4*)(o + (up ? 16 : 0)) = up ? hi : lo;
      *(u32x4*)(o + (up ? 0 : 16)) = up ? lo : hi;
    }
  };

  // a lane's place in a transposing read: token 8 g + i / 4 (and 4 on), 4 columns of the pair
  const int at = ((8 * g + (i >> 2)) * 128 + (i & 3) * 8) | ((((i >> 3) & 1) | ((g & 1) << 1)) << 5);
  const char* const pd = sm + w * kBlk;
  const char* const px = sm + kX + group * 2 * kBlk;
  bf16x8 fd[2][FN], fx[2][FM];
  f32x4 acc[FM][FN];
  float sums[FN] = {0.f, 0.f, 0.f, 0.f};   // of this lane's tokens of column i of each fragment
#pragma unroll
  for (int m = 0; m < FM; ++m)
#pragma unroll
    for (int f = 0; f < FN; ++f) acc[m][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto read_step = [&](int s, auto with_dy) __attribute__((always_inline)) {   // and the copies, between the reads
    auto read = [&](const char* p, int pair) __attribute__((always_inline)) {
      const char* q = p + (at ^ (pair << 5));
      union { i16x4 h[2]; bf16x8 v; } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)q);
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(q + 512));
      return u.v;
    };
    static_for<0, 2 * (FN + FM)>([&](auto jc) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value, h = j / (FN + FM), r = j % (FN + FM);
      if constexpr (r < FN) fd[h][r] = read(pd + (s & 1) * 4 * kBlk + h * 4096, r);
      else fx[h][r - FN] = read(px + ((r - FN) >> 2) * kBlk + h * 4096, (r - FN) & 3);
      if constexpr (decltype(with_dy)::value && j % 2 == 0 && j < 16) copy_dy(std::integral_constant<int, j / 2>{});
      if constexpr (j % 2 == 1 && j >= 17 && j < 23) copy_codes(std::integral_constant<int, (j - 17) / 2>{});
      __builtin_amdgcn_sched_barrier(0);
    });
    __builtin_amdgcn_sched_barrier(0);
  };
  auto multiply = [&](int s) __attribute__((always_inline)) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < FM; ++m)
#pragma unroll
        for (int f = 0; f < FN; ++f)
          acc[m][f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[h][m], fd[h][f], acc[m][f], 0, 0, 0);
    if (group == 0 && a.db && s % a.tiles_k == tk) {
#pragma unroll
      for (int f = 0; f < FN; ++f)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const bf16x8 d = fd[h][f];
          sums[f] += (((float)d[0] + (float)d[1]) + ((float)d[2] + (float)d[3])) +
                     (((float)d[4] + (float)d[5]) + ((float)d[6] + (float)d[7]));
        }
    }
    __builtin_amdgcn_s_setprio(0);
  };
  auto turn = []() __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
#define FVSR_WAIT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")
#define FVSR_READ_DONE() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")

  if (group == 0) static_for<0, 8>(copy_dy);
  for (int s = 0; s < 2; ++s) {
    static_for<0, 3>(copy_codes);
    next_codes();
  }
  FVSR_WAIT(0);
  if (group == 1) {
    read_codes(0);
    FVSR_READ_DONE();
    widen();
    static_for<0, 3>(copy_codes);
    next_codes();
  }
  turn();
  if (group == 1) turn();   // phase 0
  for (int s = 0; s < steps; ++s) {
    if (group == 0) {
      FVSR_WAIT(11);        // codes of s; asked for since: dY(s), codes of s + 1
      read_codes(s);
      next_dy();
      FVSR_READ_DONE();     // their place is free
      widen();
      read_step(s, std::true_type{});
      next_codes();
    } else {
      FVSR_WAIT(3);         // codes of s + 1; since: codes of s + 2
      read_codes(s + 1);
      FVSR_READ_DONE();
      widen();
      read_step(s, std::false_type{});
      next_codes();
    }
    turn();
    multiply(s);
    if (group == 0) FVSR_WAIT(3);   // dY(s + 1); since: codes of s + 2
    if (group == 0 || s + 1 < steps) turn();
  }
  FVSR_WAIT(0);             // copies (of zeros) into this workgroup's LDS
#undef FVSR_WAIT
#undef FVSR_READ_DONE

#pragma unroll
  for (int f = 0; f < FN; ++f) {   // over the lanes (g, i) of a column
    sums[f] += __shfl_xor(sums[f], 16);
    sums[f] += __shfl_xor(sums[f], 32);
  }
  O* dw = (O*)a.dw + (int64_t)blockIdx.y * a.N * a.K;
#pragma unroll
  for (int f = 0; f < FN; ++f) {
    const int n = n0 + 16 * f + i;
    if (n >= a.N) continue;
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int c = k0 + group * 128 + 16 * m + 4 * g;
      store4(dw + (int64_t)n * a.K + c, acc[m][f], a.K - c);
    }
    if (group == 0 && a.db && g == 0) a.db[((int64_t)blockIdx.y * a.tiles_k + tk) * a.N + n] = sums[f];
  }
}

// rows of N elements, N not a multiple of 8, to rows of N rounded up to one (the rest zeros)
__global__ __launch_bounds__(256) void pad_rows_kernel(const bf16* __restrict__ in, int64_t rows, int N, bf16* __restrict__ out) {
  const int vectors = (N + 7) / 8;
  const int64_t n = rows * vectors;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / vectors;
    const int c = (int)(i - row * vectors) * 8;
    const bf16* p = in + row * N + c;
    u32x4 v = u32x4{0, 0, 0, 0};
    if (c + 8 <= N) {
      v = *(const any16*)p;
    } else {
      bf16* d = (bf16*)&v;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < N) d[e] = p[e];
    }
    ((u32x4*)out)[i] = v;
  }
}

// dw = the sum over parts of their (N, K) partial results, in order (zeros if there are none), by the first `blocks`
// workgroups; the others, if any, add up `sums` partial column sums, 64 columns each, a fourth of them a wave
template <typename O>
__global__ __launch_bounds__(256) void weight_grad_join_kernel(const float* __restrict__ part, int parts, int64_t n,
                                                               O* __restrict__ dw, int blocks,
                                                               const float* __restrict__ col, int sums, int N,
                                                               float* __restrict__ db) {
  if ((int)blockIdx.x >= blocks) {
    __shared__ float sm[4][64];
    const int l = threadIdx.x & 63, q = threadIdx.x >> 6, c = ((int)blockIdx.x - blocks) * 64 + l;
    float s = 0.f;
    if (c < N)
#pragma unroll 4
      for (int p = q; p < sums; p += 4) s += col[(int64_t)p * N + c];
    sm[q][l] = s;
    __syncthreads();
    if (q == 0 && c < N) db[c] = (sm[0][l] + sm[1][l]) + (sm[2][l] + sm[3][l]);
    return;
  }
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (int64_t)blocks * 1024) {
    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
    const int have = (int)min((int64_t)4, n - i);
    for (int p = 0; p < parts; ++p) {
      const float* from = part + p * n + i;
      if (have == 4) s += *(const any_f32x4*)from;
      else
        for (int e = 0; e < have; ++e) s[e] += from[e];
    }
    store4(dw + i, s, have);
  }
}

int launch_param_sum(const float* part, int parts, int n, int split, float* out, float* out2, hipStream_t stream);   // rows8.hip

// How a weight gradient is cut up: the tokens of a tile into parts of at least kMinSteps steps, by what the whole
// takes: rounds of 256 workgroups, of 1.6 us a step and 6 us to start and end one, then the parts' sums at the copy's
// rate. As many as fill the card, or up to 4 that even out a ragged last round, if that gains a twelfth (4096 x 4608,
// 288 tiles: 17280 tokens 844 us whole, 659 in 3 parts; 2048 117, 142 in 2: whole. 1400 x 5700, 138 tiles, 17280
// tokens: 515, 415 in 3). Rows of dY that are not whole 16 bytes, which the copies into LDS need, are copied to such
// first (4000 x 1536 x 4500: 90 us; tiles of 128 that read them as they are, without such copies, 310).
struct WeightGradPlan {
  bool pad;
  int tiles_n, tiles_k, parts;
  int64_t part_rows;
  int sum_parts;   // partial column sums
};
constexpr int kMinSteps = 4;
static WeightGradPlan weight_grad_plan(int64_t rows, int N, int K) {
  WeightGradPlan p;
  p.pad = N % 8 != 0;
  p.tiles_n = (int)ceil_div(N, 256);
  p.tiles_k = (int)ceil_div(K, 256);
  const int64_t tiles = (int64_t)p.tiles_n * p.tiles_k, steps = ceil_div(rows, 64);
  const int64_t most = std::max<int64_t>(1, steps / kMinSteps);
  auto ns = [&](int64_t parts) {
    return ceil_div(tiles * parts, 256) * (ceil_div(steps, parts) * 1600 + 6000) + (parts > 1 ? parts * N * K / 600 + 3000 : 0);
  };
  const int64_t fill = std::min(most, std::max<int64_t>(1, 256 / tiles));
  int64_t parts = fill;
  for (int64_t p = 1; p <= std::min<int64_t>(4, most); ++p)
    if (ns(p) < ns(parts)) parts = p;
  if (ns(parts) * 12 > ns(fill) * 11) parts = fill;
  p.part_rows = ceil_div(steps, parts) * 64;
  p.parts = rows > 0 ? (int)ceil_div(rows, p.part_rows) : 0;
  p.sum_parts = p.parts * p.tiles_k;
  return p;
}
// the workspace: partial column sums, partial products, the copy of dY, each 16-byte aligned
struct WeightGradSpace {
  size_t part, dy, bytes;
};
static WeightGradSpace weight_grad_space(const WeightGradPlan& p, int64_t rows, int N, int K) {
  auto up = [](size_t n) { return (n + 15) & ~size_t(15); };
  WeightGradSpace s;
  s.part = up((size_t)p.sum_parts * N * sizeof(float));
  s.dy = s.part + (p.parts > 1 ? up((size_t)p.parts * N * K * sizeof(float)) : 0);
  s.bytes = s.dy + (p.pad ? (size_t)rows * ceil_div(N, 8) * 16 : 0);
  return s;
}
size_t weight_grad_workspace(int64_t rows, int N, int K) {
  return weight_grad_space(weight_grad_plan(rows, N, K), rows, N, K).bytes;
}

int launch_weight_grad(const void* dy, int64_t rows, int N, In8 x, int K, int out_dtype, void* dw, float* db, void* ws,
                       hipStream_t stream) {
  if (rows >= (int64_t)1 << 31) return set_error(FVSR_ERR_UNSUPPORTED, "linear8_weight_grad: too many rows");
  const WeightGradPlan p = weight_grad_plan(rows, N, K);
  const WeightGradSpace space = weight_grad_space(p, rows, N, K);
  const int64_t tiles = (int64_t)p.tiles_n * p.tiles_k;
  if (tiles >= 1 << 22) return set_error(FVSR_ERR_UNSUPPORTED, "linear8_weight_grad: too many output tiles for one launch");
  float* const sums = (float*)ws;
  float* const part = (float*)((char*)ws + space.part);
  WeightGradArgs a{};
  a.dy = (const bf16*)dy; a.ld = N; a.x = x; a.rows = rows; a.part_rows = p.part_rows;
  a.N = N; a.K = K; a.runs = runs_of(K); a.ss = scale_stride(K);
  a.dw = p.parts > 1 ? part : dw;
  a.db = db ? sums : nullptr;
  a.tiles_n = p.tiles_n;
  a.tiles_k = p.tiles_k;
  const bool wide = p.parts > 1 || out_dtype == FVSR_DTYPE_F32;
  const dim3 grid((unsigned)tiles, (unsigned)p.parts);
  if (p.parts > 0 && p.pad) {
    a.ld = (int)ceil_div(N, 8) * 8;
    a.dy = (const bf16*)((char*)ws + space.dy);
    const int64_t blocks = ceil_div(rows * (a.ld / 8), 256);
    hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(256), 0, stream,
                       (const bf16*)dy, rows, N, (bf16*)((char*)ws + space.dy));
    FVSR_HIP_CHECK(hipGetLastError());
  }
  if (p.parts > 0) {
    if (wide) hipLaunchKernelGGL((weight_grad_kernel<float>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((weight_grad_kernel<bf16>), grid, dim3(512), 0, stream, a);
    FVSR_HIP_CHECK(hipGetLastError());
  }
  if (p.parts != 1) {   // also no token: zeros
    const int64_t n = (int64_t)N * K;
    const int blocks = (int)std::min<int64_t>(ceil_div(n, 1024), 1 << 20);
    const dim3 join((unsigned)(blocks + (db ? ceil_div(N, 64) : 0)));
    if (out_dtype == FVSR_DTYPE_F32)
      hipLaunchKernelGGL((weight_grad_join_kernel<float>), join, dim3(256), 0, stream, part, p.parts, n, (float*)dw, blocks,
                         sums, p.sum_parts, N, db);
    else
      hipLaunchKernelGGL((weight_grad_join_kernel<bf16>), join, dim3(256), 0, stream, part, p.parts, n, (bf16*)dw, blocks,
                         sums, p.sum_parts, N, db);
    FVSR_HIP_CHECK(hipGetLastError());
    return FVSR_OK;
  }
  if (!db) return FVSR_OK;
  return launch_param_sum(sums, p.sum_parts, N, N, db, nullptr, stream);
}

}  // namespace fvsr
