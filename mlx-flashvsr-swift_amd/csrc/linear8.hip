// Products with 8-bit operands for gfx950 (MI355X): the linear layer y = x W^T + b (+ GELU) from 8-bit tokens and weights, and
// its weight gradient dW = dY^T X from bf16 gradients and the 8-bit tokens that the layer read.
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
// 16 (or 4) bytes a lane from a buffer straight into LDS at `lds` + 16 (4) * lane; what lies past the buffer's end is stored as
// 0. The copy is waited for with vmcnt. One wait state has to pass between the write of M0 and its use, hence the s_nop.
__device__ __forceinline__ void copy16(u32x4 rsrc, uint32_t lds, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc));
}
__device__ __forceinline__ void copy4(u32x4 rsrc, uint32_t lds, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(rsrc));
}

struct Linear8Args {
  In8 x, w;
  int64_t rows;
  int N, runs, ss;       // output features; runs and scale bytes a row of both operands
  const void* bias;      // may be null
  int bias_f32, gelu, vec_out;
  void* y;
  int tiles_m, tiles_n;
};

// 0.5 y (1 + tanh(sqrt(2 / pi) (y + 0.044715 y^3))) = y / (1 + exp(-2 sqrt(2 / pi) (y + 0.044715 y^3))), the exponential in base 2:
// its argument overflows to +inf (the result then is 0) only where y is far below zero
__device__ __forceinline__ float gelu_tanh(float y) {
  constexpr float k = -2.f * 0.7978845608028654f * 1.4426950408889634f;
  const float e = __builtin_amdgcn_exp2f(k * y * fmaf(0.044715f * y, y, 1.f));
  return y * __builtin_amdgcn_rcpf(1.f + e);
}

// Tile of TN output features x TM tokens, WN x WM waves; a step is one run: 128 codes of every row, and their scales in the
// matrix instruction.
//
// v_mfma_scale_f32_16x16x128_f8f6f4 D (16 x 16) += A (16 x 128) B (128 x 16): lane l gives 32 codes of row l % 16 of A and of
// column l % 16 of B, and the scale byte of its 32 codes, taken from byte OP of a register; all of a run have one scale, so which 32
// codes go with which lane does not matter as long as A and B agree. A is the weights: a lane's 4 results are then 4 features of
// one token. Fragment f of a wave holds the features 32 (f / 2) + 8 (i / 4) + 4 (f % 2) + i % 4, i = 0 .. 15, so that two fragments
// leave a lane 8 adjacent features: 16-byte stores, 64 bytes a token and instruction.
//
// LDS holds two steps: rows of 128 bytes, the 16-byte chunks XOR-ed by a number of the row under which the 16 rows that one
// instruction reads fall on 16 places of the 64 banks; copies go from memory to LDS directly (the XOR is on the source side), the
// next step's while this one's products run. A word of scales holds 4 steps.
template <int TN, int TM, int WN, int WM, typename O>
__global__ __launch_bounds__(64 * WN * WM, 2) void linear8_kernel(Linear8Args a) {
  constexpr int kWaves = WN * WM, FN = TN / WN / 16, FM = TM / WM / 16;
  static_assert(FN % 2 == 0 && (TN + TM) % (8 * kWaves) == 0 && (TN + TM) % 64 == 0, "tile");
  constexpr int kStage = (TN + TM) * kRun, kScales = (TN + TM) * 4;
  __shared__ __align__(1024) char sm[2 * kStage + 2 * kScales];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // tiles: every XCD a contiguous range, ordered in bands of 8 tiles of tokens so that a band's codes and the weights stay in its L2
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

  auto swz_w = [](int r) { return ((r >> 1) & 1) | (((r >> 3) & 3) << 1); };
  auto swz_x = [](int r) { return (r >> 1) & 7; };
  auto copy_step = [&](int k) {
    const uint32_t base = lds0 + (k & 1) * kStage;
    static_for<0, (TN + TM) / (8 * kWaves)>([&](auto ic) {
      const int r8 = (decltype(ic)::value * kWaves + wave) * 8;   // 8 rows a wave and copy
      const int r = r8 + (lane >> 3), c = lane & 7;
      if (r8 < TN)
        copy16(rw, base + r8 * kRun, (uint32_t)(r * ld + k * kRun + ((c ^ swz_w(r)) << 4)));
      else
        copy16(rx, base + r8 * kRun, (uint32_t)((r - TN) * ld + k * kRun + ((c ^ swz_x(r - TN)) << 4)));
    });
    if ((k & 3) == 0) {
      const uint32_t sbase = lds0 + 2 * kStage + ((k >> 2) & 1) * kScales;
#pragma unroll
      for (int r64 = wave * 64; r64 < TN + TM; r64 += kWaves * 64) {
        const int r = r64 + lane;
        if (r64 < TN) copy4(sw, sbase + r64 * 4, (uint32_t)(r * a.ss + k));
        else copy4(sx, sbase + r64 * 4, (uint32_t)((r - TN) * a.ss + k));
      }
    }
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

  copy_step(0);
  int qw[FN], qx[FM];
  for (int k0 = 0; k0 < a.runs; k0 += 4) {
    static_for<0, 4>([&](auto kc) {
      constexpr int OP = decltype(kc)::value;
      const int k = k0 + OP;
      if (k >= a.runs) return;
      wait_all_and_sync();   // step k is in LDS, and nobody reads step k - 1 any more
      if (k + 1 < a.runs) copy_step(k + 1);
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

  O* y = (O*)a.y;
#pragma unroll
  for (int p = 0; p < FN / 2; ++p) {
    const int n = n0 + wn * (TN / WN) + 32 * p + 8 * g;
    float b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      b[e] = !a.bias || n + e >= a.N ? 0.f : a.bias_f32 ? ((const float*)a.bias)[n + e] : (float)((const bf16*)a.bias)[n + e];
#pragma unroll
    for (int m = 0; m < FM; ++m) {
      const int64_t row = m0 + rx0 + 16 * m;
      if (row >= a.rows) continue;
      O v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float s = acc[2 * p + (e >> 2)][m][e & 3] + b[e];
        if (a.gelu) s = gelu_tanh(s);
        v[e] = (O)s;
      }
      O* out = y + row * a.N + n;
      if (a.vec_out && n + 8 <= a.N) {
        *(u32x4*)out = *(u32x4*)v;
        if constexpr (sizeof(O) == 4) ((u32x4*)out)[1] = ((u32x4*)v)[1];
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < a.N) out[e] = v[e];
      }
    }
  }
}

size_t linear8_workspace(int64_t, int, int) { return 0; }

int launch_linear8(In8 x, int64_t rows, int K, In8 w, int N, int bias_dtype, const void* bias, int gelu, int out_dtype,
                   void* y, void*, hipStream_t stream) {
  if (rows <= 0) return FVSR_OK;
  Linear8Args a{};
  a.x = x; a.w = w; a.rows = rows; a.N = N; a.runs = runs_of(K); a.ss = scale_stride(K);
  a.bias = bias; a.bias_f32 = bias_dtype == FVSR_DTYPE_F32; a.gelu = gelu; a.y = y;
  a.vec_out = rows_vectorize(y, N);
  constexpr int TN = 128, TM = 128;
  a.tiles_m = (int)ceil_div(rows, TM);
  a.tiles_n = (int)ceil_div(N, TN);
  const int64_t tiles = ceil_div(rows, TM) * a.tiles_n;
  if (tiles >= 1 << 24) return set_error(FVSR_ERR_UNSUPPORTED, "linear8: too many output tiles for one launch");
  if (out_dtype == FVSR_DTYPE_BF16)
    hipLaunchKernelGGL((linear8_kernel<TN, TM, 2, 2, bf16>), dim3((unsigned)tiles), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((linear8_kernel<TN, TM, 2, 2, float>), dim3((unsigned)tiles), dim3(256), 0, stream, a);
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

// ------------------------------------------------------------------------------------------------------------
// weight gradient
// ------------------------------------------------------------------------------------------------------------
struct WeightGradArgs {
  const bf16* dy;
  In8 x;
  int64_t rows;
  int N, K, runs, ss;
  int vec_dy, vec_out;
  void* dw;
  int tiles_n, tiles_k;
};

// dW (N, K) = dY^T X: a tile of TN x TK, steps of 32 tokens. Both operands lie token-major, so the product's depth runs across rows:
// the tiles are stored in LDS as they come, [token][column] in bf16 (codes times scales are exact in bf16), and
// ds_read_b64_tr_b16 hands a lane 4 tokens of one column: 16 lanes read 4 rows of 16 columns, lane i gets column i of the four.
template <int TN, int TK, int WN, int WK, typename O>
__global__ __launch_bounds__(64 * WN * WK, 2) void weight_grad_kernel(WeightGradArgs a) {
  constexpr int kThreads = 64 * WN * WK, kTokens = 32, FN = TN / WN / 16, FK = TK / WK / 16;
  constexpr int kDy = kTokens * TN / 8 / kThreads, kX = kTokens * TK / 8 / kThreads;   // 8-element vectors a thread
  static_assert(kDy > 0 && kX > 0, "tile");
  __shared__ __align__(1024) char sm[2][kTokens * (TN + TK) * 2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = xcd_remap(blockIdx.x, gridDim.x);
  const int tk = t % a.tiles_k, tn = t / a.tiles_k;
  const int n0 = tn * TN, k0 = tk * TK;

  u32x4 rdy[kDy];
  uint2 rx[kX];
  uint32_t rs[kX];
  auto load = [&](int64_t m0) {
#pragma unroll
    for (int j = 0; j < kDy; ++j) {
      const int v = j * kThreads + threadIdx.x, r = v / (TN / 8), c = n0 + v % (TN / 8) * 8;
      const int64_t row = m0 + r;
      rdy[j] = u32x4{0, 0, 0, 0};
      if (row < a.rows) {
        const bf16* p = a.dy + row * a.N + c;
        if (a.vec_dy) {
          if (c < a.N) rdy[j] = *(const u32x4*)p;
        } else {
          bf16* d = (bf16*)&rdy[j];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (c + e < a.N) d[e] = p[e];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < kX; ++j) {
      const int v = j * kThreads + threadIdx.x, r = v / (TK / 8), c = k0 + v % (TK / 8) * 8;
      const int64_t row = m0 + r;
      rx[j] = make_uint2(0, 0);
      rs[j] = 0;
      if (row < a.rows && c < a.runs * kRun) {
        rx[j] = *(const uint2*)(a.x.codes + row * (int64_t)a.runs * kRun + c);
        rs[j] = a.x.scales[row * a.ss + c / kRun];
      }
    }
  };
  auto put = [&](char* s) {
#pragma unroll
    for (int j = 0; j < kDy; ++j) {
      const int v = j * kThreads + threadIdx.x, r = v / (TN / 8), c = v % (TN / 8) * 8;
      *(u32x4*)(s + (r * TN + c) * 2) = rdy[j];
    }
#pragma unroll
    for (int j = 0; j < kX; ++j) {
      const int v = j * kThreads + threadIdx.x, r = v / (TK / 8), c = v % (TK / 8) * 8;
      const float by = __uint_as_float(rs[j] << 23);
      bf16x2 q[4];
      q[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rx[j].x, by, false);
      q[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rx[j].x, by, true);
      q[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rx[j].y, by, false);
      q[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(rx[j].y, by, true);
      *(u32x4*)(s + kTokens * TN * 2 + (r * TK + c) * 2) = *(u32x4*)q;
    }
  };

  const int wn = wave % WN, wk = wave / WN, i = lane & 15, g = lane >> 4;
  f32x4 acc[FK][FN];
#pragma unroll
  for (int f = 0; f < FK; ++f)
#pragma unroll
    for (int n = 0; n < FN; ++n) acc[f][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  load(0);
  int turn = 0;
  for (int64_t m0 = 0; m0 < a.rows; m0 += kTokens, turn ^= 1) {
    put(sm[turn]);
    __syncthreads();
    if (m0 + kTokens < a.rows) load(m0 + kTokens);
    // lane (g, i): tokens 8 g .. 8 g + 7 of column i of a fragment
    auto read = [&](const char* s, int width, int col) {
      const char* p = s + ((8 * g + (i >> 2)) * width + col + (i & 3) * 4) * 2;
      union { i16x4 h[2]; bf16x8 v; } u;
      u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)p);
      u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(p + 4 * width * 2));
      return u.v;
    };
    bf16x8 fn[FN];
#pragma unroll
    for (int n = 0; n < FN; ++n) fn[n] = read(sm[turn], TN, wn * (TN / WN) + 16 * n);
#pragma unroll
    for (int f = 0; f < FK; ++f) {
      const bf16x8 fk = read(sm[turn] + kTokens * TN * 2, TK, wk * (TK / WK) + 16 * f);
#pragma unroll
      for (int n = 0; n < FN; ++n) acc[f][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fk, fn[n], acc[f][n], 0, 0, 0);
    }
  }
  O* dw = (O*)a.dw;
#pragma unroll
  for (int n = 0; n < FN; ++n) {
    const int row = n0 + wn * (TN / WN) + 16 * n + i;
    if (row >= a.N) continue;
#pragma unroll
    for (int f = 0; f < FK; ++f) {
      const int c = k0 + wk * (TK / WK) + 16 * f + 4 * g;
      O* out = dw + (int64_t)row * a.K + c;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c + e < a.K) out[e] = (O)acc[f][n][e];
    }
  }
}

// partial column sums of dy: workgroup (x, y) adds rows y, y + gridDim.y, .. of 4 waves' worth of 64 columns each
__global__ __launch_bounds__(256) void column_sum_kernel(const bf16* __restrict__ dy, int64_t rows, int N, float* __restrict__ part) {
  __shared__ float sm[256];
  const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
  float s = 0.f;
  if (c < N)
    for (int64_t r = (int64_t)blockIdx.y * 4 + q; r < rows; r += (int64_t)gridDim.y * 4) s += (float)dy[r * N + c];
  sm[threadIdx.x] = s;
  __syncthreads();
  if (q == 0 && c < N)
    part[(int64_t)blockIdx.y * N + c] = (sm[threadIdx.x] + sm[64 + threadIdx.x]) + (sm[128 + threadIdx.x] + sm[192 + threadIdx.x]);
}

int launch_param_sum(const float* part, int parts, int64_t stride, int n, float* out, hipStream_t stream);

constexpr int kSumParts = 64;
size_t weight_grad_workspace(int64_t rows, int N, int K) {
  (void)rows; (void)K;
  return (size_t)kSumParts * N * sizeof(float);
}

int launch_weight_grad(const void* dy, int64_t rows, int N, In8 x, int K, int out_dtype, void* dw, float* db, void* ws,
                       hipStream_t stream) {
  WeightGradArgs a{};
  a.dy = (const bf16*)dy; a.x = x; a.rows = rows; a.N = N; a.K = K; a.runs = runs_of(K); a.ss = scale_stride(K);
  a.vec_dy = rows_vectorize(dy, N);
  a.dw = dw;
  constexpr int TN = 128, TK = 128;
  a.tiles_n = (int)ceil_div(N, TN);
  a.tiles_k = (int)ceil_div(K, TK);
  const int64_t tiles = (int64_t)a.tiles_n * a.tiles_k;
  if (tiles >= 1 << 24) return set_error(FVSR_ERR_UNSUPPORTED, "linear8: too many output tiles for one launch");
  if (out_dtype == FVSR_DTYPE_BF16)
    hipLaunchKernelGGL((weight_grad_kernel<TN, TK, 2, 2, bf16>), dim3((unsigned)tiles), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((weight_grad_kernel<TN, TK, 2, 2, float>), dim3((unsigned)tiles), dim3(256), 0, stream, a);
  FVSR_HIP_CHECK(hipGetLastError());
  if (!db) return FVSR_OK;
  const int parts = (int)std::max<int64_t>(1, std::min<int64_t>(kSumParts, ceil_div(rows, 16)));
  hipLaunchKernelGGL(column_sum_kernel, dim3((unsigned)ceil_div(N, 64), parts), dim3(256), 0, stream, a.dy, rows, N, (float*)ws);
  FVSR_HIP_CHECK(hipGetLastError());
  return launch_param_sum((const float*)ws, parts, N, N, db, stream);
}

}  // namespace fvsr
