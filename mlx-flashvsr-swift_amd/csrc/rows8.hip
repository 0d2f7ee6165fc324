// Row operators next to the 8-bit products, for gfx950 (MI355X): tokens to 8 bits and back, and layer norm with its
// gradient, which write and read the 8-bit form in the passes that hold the row anyway.
//
//   y  = n w + b,  n = (x - mean) rstd,  rstd = 1 / sqrt(var + eps)      (mean and var over the row's C channels)
//   dx = rstd (g - mean(g) - n mean(g n)),  g = dy w
//   dw = sum over rows of dy n,  db = sum over rows of dy
//
// All of them move each row once and compute a few operations a channel: memory-bound. A row's channels stay in
// registers between the passes over it (sums, then squares, then the result), in 32 bits.
//
// bf16, against 4.8 TB/s that a copy of 4 GB reaches here, over buffers of more than the memory-side cache: 17280 x
// 1536 norm 26.4 us (106 MB, 4.0 TB/s; 21.3 where each pass writes the same output, part of which stays in that cache),
// with its statistics and x in 8 bits 30.5 (133 MB, 4.3), to 8 bits 24.1 (80 MB, 3.3; 30-33 right behind a product
// whose output still drains), gradient from 8 bits 27.4 (133 MB, 4.9) and 5-6 to add the parts; 17280 x 8960 quantize
// 84-95 us (466 MB, 4.9-5.5), dequantize 75-81 (5.7-6.2). One row of 1536: 3.0 us, a chain of two round trips.
#include <algorithm>

#include "blocks8.hpp"

namespace fvsr {

struct NormArgs {
  const void* x;
  int64_t rows;
  int C;
  float eps;
  const void *w, *b;   // either may be null
  void* y;             // null: not written
  Out8 y8, x8;         // codes null: not written
  float* stats;        // (rows, 2) mean, rstd; may be null
};

struct NormGradArgs {
  const void *dy, *x;   // x null: read from x8
  In8 x8;
  const float* stats;
  int64_t rows;
  int C;
  const void* w;        // may be null
  void* dx;
  float* part;          // (blocks, 2, C) partial dw and db; null: neither is made
};

// the sum over a wave (every lane active), by DPP rotations within its rows of 16 lanes and a lane of each row: no LDS
// round trips
__device__ __forceinline__ float wave_sum(float x) {
  auto rot = [](float v, auto ctrl) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  x += rot(x, std::integral_constant<int, 0x128>{});   // row_ror:8
  x += rot(x, std::integral_constant<int, 0x124>{});
  x += rot(x, std::integral_constant<int, 0x122>{});
  x += rot(x, std::integral_constant<int, 0x121>{});
  auto row = [&](int r) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16 * r)); };
  return (row(0) + row(1)) + (row(2) + row(3));
}

// sums over the WAVES waves that share a row, in a fixed order; `sm` holds 2 * WAVES floats, which a wave may
// still read when another has left the call: successive calls alternate between two areas
template <int WAVES>
__device__ __forceinline__ void team_sum2(float& a, float& b, float* sm) {
  a = wave_sum(a);
  b = wave_sum(b);
  if constexpr (WAVES > 1) {
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
      sm[2 * wave] = a;
      sm[2 * wave + 1] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      a += sm[2 * w];
      b += sm[2 * w + 1];
    }
  }
}

// One row a team of WAVES waves (a workgroup holds max(WAVES, 4) waves), NV vectors of 8 channels a lane: lane L of the
// team and vector j hold 8 channels of run 4 * WAVES * j + L / 16.
template <typename T, typename P, bool EIGHTS, int WAVES, int NV>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void layer_norm_kernel(NormArgs a) {
  __shared__ float sm[2][2 * WAVES];
  const int l16 = threadIdx.x & 15, C = a.C;
  const int64_t row = WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x;
  if (row >= a.rows) return;   // WAVES > 1: never (one row a workgroup)
  const int run0 = (WAVES == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x) >> 4;
  const T* x = (const T*)a.x + row * C;
  const int runs = runs_of(C), ss = scale_stride(C);
  float v[NV][8];
  float sum = 0.f, none = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    load8<T, EIGHTS>(x, (run0 + 4 * WAVES * j) * kRun, l16, C, v[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += v[j][e];
  }
  team_sum2<WAVES>(sum, none, sm[0]);
  const float mean = sum / (float)C;
  if (a.x8.codes) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int run = run0 + 4 * WAVES * j;
      uint32_t s;
      const uint2 c = encode8(v[j], s);
      if (run < runs) store_codes(a.x8.codes + (row * runs + run) * kRun, l16, c);
      if (run < ss && l16 == 0) a.x8.scales[row * ss + run] = run < runs ? (uint8_t)s : 0;
    }
  }
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c0 = (run0 + 4 * WAVES * j) * kRun;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[j][e] = c0 + l16 * 8 + e < C ? v[j][e] - mean : 0.f;
      sq = fmaf(v[j][e], v[j][e], sq);
    }
  }
  team_sum2<WAVES>(sq, none, sm[1]);
  const float rstd = 1.f / sqrtf(sq / (float)C + a.eps);
  if (a.stats && (WAVES == 1 ? threadIdx.x & 63 : threadIdx.x) == 0) {
    a.stats[2 * row] = mean;
    a.stats[2 * row + 1] = rstd;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int run = run0 + 4 * WAVES * j;
    float w[8], b[8], y[8];
    if (a.w) load8<P, EIGHTS>((const P*)a.w, run * kRun, l16, C, w);
    if (a.b) load8<P, EIGHTS>((const P*)a.b, run * kRun, l16, C, b);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = v[j][e] * rstd;
      if (a.w) y[e] *= w[e];
      if (a.b) y[e] += b[e];
      if (run * kRun + l16 * 8 + e >= C) y[e] = 0.f;   // also where the row's rstd is not finite
    }
    if (a.y) store8<T, EIGHTS>((T*)a.y + row * C, run * kRun + l16 * 8, 0, C, y);
    if (a.y8.codes) {
      uint32_t s;
      const uint2 c = encode8(y, s);
      if (run < runs) store_codes(a.y8.codes + (row * runs + run) * kRun, l16, c);
      if (run < ss && l16 == 0) a.y8.scales[row * ss + run] = run < runs ? (uint8_t)s : 0;
    }
  }
}

// The gradient: teams walk over the rows (the grid is a fixed number of workgroups) and keep their part of dw and db in
// registers; the workgroup's sum goes to `part`, and param_sum_kernel adds the workgroups' up: no atomics, the same
// result every time. Where C is not a multiple of 8 (not EIGHTS), the lane of the row's end takes its last 8 channels,
// and skips the first `dup` of them, which its neighbour has too: one load, which nothing waits for before its row is
// worked on.
template <typename T, typename P, bool EIGHTS, int WAVES, int NV, bool X8>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES, EIGHTS && WAVES < 16 ? 2 : 1)
void layer_norm_grad_kernel(NormGradArgs a) {
  __shared__ float sm[2][2 * WAVES];
  __shared__ float join[WAVES == 1 ? 4 * 64 * 16 : 1];
  const int l16 = threadIdx.x & 15, lane = threadIdx.x & 63, C = a.C;
  const int team = WAVES == 1 ? (int)(threadIdx.x >> 6) : 0, teams = WAVES == 1 ? 4 : 1;
  const int run0 = (WAVES == 1 ? lane : (int)threadIdx.x) >> 4;
  const int runs = runs_of(C), ss = scale_stride(C);
  float w[NV][8], dw[NV][8], db[NV][8];
  auto first = [&](int j) { return (run0 + 4 * WAVES * j) * kRun + l16 * 8; };   // the lane's channels of vector j
  auto held = [&](int j) { return EIGHTS ? first(j) : min(first(j), max(0, C - 8)); };
  auto dup = [&](int j) { return first(j) - held(j); };                          // 8 or more past the row's end
  auto load_held = [&](auto* p, int j) {
    using E = std::remove_cv_t<std::remove_reference_t<decltype(*p)>>;
    Raw8<E> r;
    u32x4* const to = (u32x4*)r.v;
    to[0] = u32x4{0, 0, 0, 0};
    if constexpr (sizeof(E) == 4) to[1] = u32x4{0, 0, 0, 0};
    if (first(j) >= C) return r;
    if (EIGHTS || C >= 8) {
      to[0] = *(const any16*)(p + held(j));
      if constexpr (sizeof(E) == 4) to[1] = *(const any16*)(p + held(j) + 4);
    } else {
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < C) r.v[e] = p[e];
    }
    return r;
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Raw8<P> rw = a.w ? load_held((const P*)a.w, j) : Raw8<P>{};
#pragma unroll
    for (int e = 0; e < 8; ++e) w[j][e] = (float)rw.v[e];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (!a.w) w[j][e] = 1.f;
      dw[j][e] = db[j][e] = 0.f;
    }
  }
  // the next row is on its way while one is worked on
  Raw8<T> rdy[NV], rx[NV];
  u32x2 rc[NV];
  uint32_t rs[NV];
  float mean = 0.f, rstd = 0.f;
  auto load = [&](int64_t row) {
    mean = a.stats[2 * row];
    rstd = a.stats[2 * row + 1];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int run = run0 + 4 * WAVES * j;
      rdy[j] = load_held((const T*)a.dy + row * C, j);
      if constexpr (X8) {
        rc[j] = u32x2{0, 0};
        if (run < runs && first(j) < C) rc[j] = *(const any8*)(a.x8.codes + row * runs * kRun + held(j));
        rs[j] = run < runs ? a.x8.scales[row * ss + run] : 0;
      } else {
        rx[j] = load_held((const T*)a.x + row * C, j);
      }
    }
  };
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * teams;
  int64_t row = (int64_t)blockIdx.x * teams + team;
  if (row < a.rows) load(row);
  for (; row < a.rows; row += step, turn ^= 1) {
    const float mu = mean, r = rstd;
    float dy[NV][8], n[NV][8];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (X8) decode8(make_uint2(rc[j][0], rc[j][1]), rs[j], n[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dy[j][e] = EIGHTS || e >= dup(j) ? (float)rdy[j].v[e] : 0.f;
        if constexpr (!X8) n[j][e] = (float)rx[j].v[e];
      }
    }
    if (row + step < a.rows) load(row + step);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      // Past the row's end dy is 0, and n has to be 0 too: the mean times rstd may pass the largest number where no
      // channel's n does. Only the last vector reaches past it; a row of less than 8 channels has no neighbour's to
      // take.
      const float m = EIGHTS && j == NV - 1 && first(j) >= C ? 0.f : mu;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        n[j][e] = (n[j][e] - m) * r;
        if (!EIGHTS && (e < dup(j) || (WAVES * NV == 1 && e >= C))) n[j][e] = 0.f;   // the neighbour's, or codes of another run
        const float g = dy[j][e] * w[j][e];
        s1 += g;
        s2 = fmaf(g, n[j][e], s2);
        dw[j][e] = fmaf(dy[j][e], n[j][e], dw[j][e]);
        db[j][e] += dy[j][e];
      }
    }
    team_sum2<WAVES>(s1, s2, sm[turn]);
    const float m1 = s1 / (float)C, m2 = s2 / (float)C;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float dx[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) dx[e] = r * (dy[j][e] * w[j][e] - m1 - n[j][e] * m2);
      store8<T, EIGHTS>((T*)a.dx + row * C, held(j), dup(j), C, dx);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    auto put = [&](float* to, int e0, f32x4 v) {   // elements e0 .. e0 + 3 of vector j
      if (first(j) + 8 <= C) {
        *(any_f32x4*)(to + held(j) + e0) = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (e0 + e >= dup(j) && held(j) + e0 + e < C) to[held(j) + e0 + e] = v[e];
      }
    };
    if constexpr (WAVES == 1) {
      // the 4 waves hold the same channels: their sums meet in LDS, [wave][16 values][lane]
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        join[(team * 16 + e) * 64 + lane] = dw[j][e];
        join[(team * 16 + 8 + e) * 64 + lane] = db[j][e];
      }
      __syncthreads();
      f32x4 s;   // values 4 team .. + 3 of lane `lane`: elements 4 (team % 2) .. + 3 of dw (team < 2) or db
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int k = 4 * team + q;
        s[q] = (join[k * 64 + lane] + join[(16 + k) * 64 + lane]) + (join[(32 + k) * 64 + lane] + join[(48 + k) * 64 + lane]);
      }
      put(part + (team < 2 ? 0 : C), 4 * (team & 1), s);
    } else {
#pragma unroll
      for (int h = 0; h < 8; h += 4) {
        put(part, h, f32x4{dw[j][h], dw[j][h + 1], dw[j][h + 2], dw[j][h + 3]});
        put(part + C, h, f32x4{db[j][h], db[j][h + 1], db[j][h + 2], db[j][h + 3]});
      }
    }
  }
}

// The sums over p < parts of part[p * n + c], c < n: columns below `split` go to out, the others to out2 (either may be
// null). 64 columns a workgroup, a sixteenth of the parts a wave, joined in a fixed order: the parts' addresses are
// known at once, so the time is that of a few loads in a row (512 parts of 2 x 1536 columns: 12 us with a quarter a
// wave).
__global__ __launch_bounds__(1024) void param_sum_kernel(const float* __restrict__ part, int parts, int n, int split,
                                                         float* __restrict__ out, float* __restrict__ out2) {
  __shared__ float sm[16][64];
  const int l = threadIdx.x & 63, c = blockIdx.x * 64 + l, q = threadIdx.x >> 6;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (c < n) {
    int p = q;
    for (; p + 48 < parts; p += 64)
#pragma unroll
      for (int u = 0; u < 4; ++u) s[u] += part[(int64_t)(p + 16 * u) * n + c];
    for (; p < parts; p += 16) s[0] += part[(int64_t)p * n + c];
  }
  sm[q][l] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  float* const to = c < split ? out : out2;
  if (q == 0 && c < n && to) {
    float t = 0.f;
#pragma unroll
    for (int u = 0; u < 16; ++u) t += sm[u][l];
    to[c < split ? c : c - split] = t;
  }
}

// A wave takes 4 runs of a row (one word of scales), 16 lanes each.
template <typename T, bool EIGHTS>
__global__ __launch_bounds__(256) void quantize_kernel(const T* __restrict__ x, int64_t rows, int C, Out8 o) {
  const int l16 = threadIdx.x & 15, r4 = (threadIdx.x & 63) >> 4;
  const int runs = runs_of(C), ss = scale_stride(C), words = ss / 4;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = unit / words;
  if (row >= rows) return;
  const int run = (int)(unit - row * words) * 4 + r4;
  float v[8];
  load8<T, EIGHTS>(x + row * C, run * kRun, l16, C, v);
  uint32_t s;
  const uint2 c = encode8(v, s);
  if (run < runs) store_codes(o.codes + (row * runs + run) * kRun, l16, c);
  if (l16 == 0) o.scales[row * ss + run] = run < runs ? (uint8_t)s : 0;
}

template <typename T, bool EIGHTS>
__global__ __launch_bounds__(256) void dequantize_kernel(In8 q, int64_t rows, int C, T* __restrict__ out) {
  const int l16 = threadIdx.x & 15, r4 = (threadIdx.x & 63) >> 4;
  const int runs = runs_of(C), ss = scale_stride(C), words = ss / 4;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t row = unit / words;
  if (row >= rows) return;
  const int run = (int)(unit - row * words) * 4 + r4;
  if (run >= runs) return;
  float v[8];
  decode8(load_codes(q.codes + (row * runs + run) * kRun, l16), q.scales[row * ss + run], v);
  store8<T, EIGHTS>(out + row * C, run * kRun + l16 * 8, 0, C, v);
}

// ------------------------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------------------------
constexpr int kMaxNormChannels = 16384;
constexpr int kGradBlocks = 512;   // two workgroups a CU

// a launch's work-items have to stay below 2^32
static int check_grid(int64_t blocks, int threads) {
  if (blocks >= (((int64_t)1 << 32) - 1) / threads) return set_error(FVSR_ERR_UNSUPPORTED, "too many rows for one launch");
  return FVSR_OK;
}

// f(waves a row, vectors a lane): one wave up to 2048 channels, 4 up to 8192, 16 up to 16384. Few waves a row share its
// work with few barriers and wave sums; many leave each lane fewer registers to hold. This rule against 4 waves from
// 1025 channels and 16 from 4097 (one or two vectors a lane): bf16 17280 x 1536 norm 26.4 us against 31.9, to 8 bits
// 24.3 against 35.9, gradient from 8 bits 27.5 against 37.7; 4000 x 8192 34.4 against 35.9, 31.9 against 38.6, 33.4
// against 34.4. It costs fp32 gradients of 4 vectors a lane, which spill 26-61 registers: 8192 x 2048 from x 62.1
// against 38.2, 4000 x 8192 119 against 73. Above 8192 channels every gradient spills 30-98 (bf16 from 8 bits, 3800 x
// 8960 104 us, 1.6 TB/s; 2000 x 16384 74, 2.2), and odd rows of 4 vectors a lane run one wave a SIMD (8000 x 2047 24.5,
// 3.4).
template <class F>
static int pick_team(int C, F&& f) {
  const int nv = (int)ceil_div(C, 512);
  if (nv <= 4) {
    switch (nv) {
      case 1: f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}); break;
      case 2: f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{}); break;
      case 3: f(std::integral_constant<int, 1>{}, std::integral_constant<int, 3>{}); break;
      default: f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{}); break;
    }
  } else if (nv <= 16) {
    switch ((nv + 3) / 4) {
      case 2: f(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{}); break;
      case 3: f(std::integral_constant<int, 4>{}, std::integral_constant<int, 3>{}); break;
      default: f(std::integral_constant<int, 4>{}, std::integral_constant<int, 4>{}); break;
    }
  } else {
    f(std::integral_constant<int, 16>{}, std::integral_constant<int, 2>{});
  }
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

// f(element type, parameter type, whether C is a multiple of 8)
template <class F>
static int pick_types(int dtype, int param_dtype, int C, F&& f) {
  auto with = [&](auto t, auto p) { return C % 8 == 0 ? f(t, p, std::true_type{}) : f(t, p, std::false_type{}); };
  if (dtype == FVSR_DTYPE_BF16) return param_dtype == FVSR_DTYPE_BF16 ? with(bf16{}, bf16{}) : with(bf16{}, float{});
  return with(float{}, float{});   // fp32 tokens take fp32 parameters
}

int max_norm_channels() { return kMaxNormChannels; }

int launch_layer_norm(int dtype, int param_dtype, const void* x, int64_t rows, int C, float eps, const void* w,
                      const void* b, void* y, Out8 y8, Out8 x8, float* stats, hipStream_t stream) {
  if (rows <= 0) return FVSR_OK;
  if (const int rc = check_grid(rows, C <= 2048 ? 64 : C <= 8192 ? 256 : 1024)) return rc;
  const NormArgs a{x, rows, C, eps, w, b, y, y8, x8, stats};
  return pick_types(dtype, param_dtype, C, [&](auto t, auto p, auto v) {
    return pick_team(C, [&](auto waves, auto nv) {
      constexpr int W = decltype(waves)::value;
      hipLaunchKernelGGL((layer_norm_kernel<decltype(t), decltype(p), decltype(v)::value, W, decltype(nv)::value>),
                         dim3((unsigned)(W == 1 ? ceil_div(rows, 4) : rows)), dim3(W == 1 ? 256 : 64 * W), 0, stream, a);
    });
  });
}

int launch_param_sum(const float* part, int parts, int n, int split, float* out, float* out2, hipStream_t stream) {
  hipLaunchKernelGGL(param_sum_kernel, dim3((unsigned)ceil_div(n, 64)), dim3(1024), 0, stream, part, parts, n, split, out, out2);
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

// a workgroup's rows are at least two for each of its teams: its parts of dw and db cost as much as a row
int64_t norm_grad_blocks(int64_t rows, int C) {
  return std::min<int64_t>(kGradBlocks, C <= 2048 ? ceil_div(rows, 8) : ceil_div(rows, 2));
}

int launch_layer_norm_grad(int dtype, int param_dtype, const void* dy, const void* x, In8 x8, const float* stats,
                           int64_t rows, int C, const void* w, void* dx, float* dw, float* db, float* part,
                           hipStream_t stream) {
  const int64_t blocks = norm_grad_blocks(rows, C);
  if (blocks > 0) {
    const NormGradArgs a{dy, x, x8, stats, rows, C, w, dx, dw || db ? part : nullptr};
    const int rc = pick_types(dtype, param_dtype, C, [&](auto t, auto p, auto v) {
      return pick_team(C, [&](auto waves, auto nv) {
        constexpr int W = decltype(waves)::value, N = decltype(nv)::value;
        constexpr bool V = decltype(v)::value;
        const dim3 grid((unsigned)blocks), block(W == 1 ? 256 : 64 * W);
        if (x8.codes)
          hipLaunchKernelGGL((layer_norm_grad_kernel<decltype(t), decltype(p), V, W, N, true>), grid, block, 0, stream, a);
        else
          hipLaunchKernelGGL((layer_norm_grad_kernel<decltype(t), decltype(p), V, W, N, false>), grid, block, 0, stream, a);
      });
    });
    if (rc) return rc;
  }
  return dw || db ? launch_param_sum(part, (int)blocks, 2 * C, C, dw, db, stream) : FVSR_OK;
}

int launch_quantize(int dtype, const void* x, int64_t rows, int C, Out8 o, hipStream_t stream) {
  if (rows <= 0) return FVSR_OK;
  const int64_t blocks = ceil_div(rows * (scale_stride(C) / 4), 4);
  if (const int rc = check_grid(blocks, 256)) return rc;
  auto go = [&](auto t, auto v) {
    using T = decltype(t);
    hipLaunchKernelGGL((quantize_kernel<T, decltype(v)::value>), dim3((unsigned)blocks), dim3(256), 0, stream, (const T*)x,
                       rows, C, o);
  };
  auto with = [&](auto t) { C % 8 == 0 ? go(t, std::true_type{}) : go(t, std::false_type{}); };
  if (dtype == FVSR_DTYPE_BF16) with(bf16{});
  else with(float{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

int launch_dequantize(In8 q, int64_t rows, int C, int dtype, void* out, hipStream_t stream) {
  if (rows <= 0) return FVSR_OK;
  const int64_t blocks = ceil_div(rows * (scale_stride(C) / 4), 4);
  if (const int rc = check_grid(blocks, 256)) return rc;
  auto go = [&](auto t, auto v) {
    using T = decltype(t);
    hipLaunchKernelGGL((dequantize_kernel<T, decltype(v)::value>), dim3((unsigned)blocks), dim3(256), 0, stream, q, rows, C,
                       (T*)out);
  };
  auto with = [&](auto t) { C % 8 == 0 ? go(t, std::true_type{}) : go(t, std::false_type{}); };
  if (dtype == FVSR_DTYPE_BF16) with(bf16{});
  else with(float{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

}  // namespace fvsr
