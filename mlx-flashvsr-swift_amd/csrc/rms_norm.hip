// Root-mean-square norm of tokens with the residual's addition before it, and its gradient, for gfx950 (MI355X).
//
//   s  = x + residual (rounded to the tokens' type, as the next layers read it; x itself without a residual)
//   y  = n w,  n = s rstd,  rstd = 1 / sqrt(mean(s^2) + eps)               (the mean over the row's C channels)
//   dx = ds + rstd (g - n mean(g n)),  g = dy w;  the same for both addends
//   dw = sum over rows of dy n
//
// Each row moves once and stays in registers between the pass that sums and the one that writes, in 32 bits: memory-bound.
// A row belongs to a team: 16 lanes up to 128 channels (a head's width), a wave, 4 or 16 waves beyond.
//
// Over sets larger than the 256 MB memory-side cache, where a copy reaches 4.7 TB/s (us, TB/s): 17280 x 1536 bf16 with residual and
// sum 45.6, 4.7; y in 8 bits 40.9, 4.6; the gradient with dw 47.6, 4.5; fp32 82.6 and 82.5, 5.1; 4000 x 8192 bf16 54, 52 and 62;
// 2000 x 16384 51, 48 and 83. One row of 1536: 3.3, a launch and two round trips.
#include <algorithm>

#include "blocks8.hpp"
#include "teams.hpp"

namespace fvsr {

int launch_param_sum(const float* part, int parts, int n, int split, float* out, float* out2, hipStream_t stream);

struct RmsArgs {
  const void* x;
  int64_t x_stride;      // elements between x's rows
  const void* r;         // residual, may be null
  int64_t rows;
  int C;
  float eps;
  const void* w;         // may be null
  void* y;               // null: not written
  Out8 y8;               // codes null: not written
  void* s;               // null: not written
  float* rstd;           // may be null
};

struct RmsGradArgs {
  const void *dy, *s;
  int64_t s_stride;
  const float* rstd;
  const void* ds;        // may be null
  int64_t rows;
  int C;
  const void* w;         // may be null
  void* dx;
  float* part;           // (blocks, C) partial dw; null: not made
};

// lanes of a team, teams of a workgroup, threads of a workgroup
template <int WAVES>
struct Team {
  static constexpr int kLanes = WAVES == 0 ? 16 : 64 * WAVES;
  static constexpr int kThreads = WAVES <= 1 ? 256 : 64 * WAVES;
  static constexpr int kTeams = kThreads / kLanes;
  static constexpr int kRuns = kLanes / 16;   // runs of 128 channels that the team's j-th vectors cover
};

// Values c0 + 8 l16 .. of a row, as load_raw8 gives them once `settle` has been called. The last part of 8 of a bf16 row is read as the
// row's last 8 values, by one load like the others, and moved into its place when it is needed: values read one by one are put together
// by waiting for them, which a row on its way ahead must not do (8000 x 4001: the gradient 94 us so, 56 at 4000).
template <typename T, bool EIGHTS>
__device__ __forceinline__ Raw8<T> load_part(const T* row, int c0, int l16, int C) {
  if (EIGHTS || sizeof(T) == 4 || C < 8) return load_raw8<T, EIGHTS>(row, c0, l16, C);
  Raw8<T> r;
  *(u32x4*)r.v = u32x4{0, 0, 0, 0};
  const int c = c0 + l16 * 8;
  if (c < C) *(u32x4*)r.v = *(const any16*)(row + min(c, C - 8));
  return r;
}
template <typename T, bool EIGHTS>
__device__ __forceinline__ void settle(Raw8<T>& r, int c0, int l16, int C) {
  if constexpr (!EIGHTS && sizeof(T) == 2) {
    const int c = c0 + l16 * 8, by = C >= 8 && c < C ? max(0, c + 8 - C) : 0;   // values too many in front
    u32x4 x = *(const u32x4*)r.v;
    if (by & 4) x = u32x4{x[2], x[3], 0, 0};
    if (by & 2) x = u32x4{x[1], x[2], x[3], 0};
    if (by & 1) x = u32x4{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16, x[2] >> 16 | x[3] << 16, x[3] >> 16};
    *(u32x4*)r.v = x;
  }
}

template <typename T, typename P, bool EIGHTS, int WAVES, int NV>
__global__ __launch_bounds__(Team<WAVES>::kThreads) void rms_norm_kernel(RmsArgs a) {
  using W = Team<WAVES>;
  __shared__ float sm[WAVES > 1 ? WAVES : 1];
  const int l16 = threadIdx.x & 15, C = a.C;
  const int64_t row = (int64_t)blockIdx.x * W::kTeams + threadIdx.x / W::kLanes;
  if (row >= a.rows) return;   // whole teams; never where a workgroup is one team
  const int run0 = (int)(threadIdx.x % W::kLanes) >> 4;
  const int runs = runs_of(C), ss = scale_stride(C);
  const T* x = (const T*)a.x + row * a.x_stride;
  Raw8<T> rx[NV], rr[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c0 = (run0 + W::kRuns * j) * kRun;
    rx[j] = load_part<T, EIGHTS>(x, c0, l16, C);
    if (a.r) rr[j] = load_part<T, EIGHTS>((const T*)a.r + row * C, c0, l16, C);
  }
  settle<T, EIGHTS>(rx[NV - 1], (run0 + W::kRuns * (NV - 1)) * kRun, l16, C);   // no vector before it is a row's last
  if (a.r) settle<T, EIGHTS>(rr[NV - 1], (run0 + W::kRuns * (NV - 1)) * kRun, l16, C);
  float v[NV][8];
  float sq = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[j][e] = (float)rx[j].v[e];
      if (a.r) v[j][e] = (float)(T)(v[j][e] + (float)rr[j].v[e]);
      sq = fmaf(v[j][e], v[j][e], sq);
    }
    if (a.s) store8<T, EIGHTS>((T*)a.s + row * C, (run0 + W::kRuns * j) * kRun + l16 * 8, 0, C, v[j]);
  }
  const float rstd = 1.f / sqrtf(team_sum<WAVES>(sq, sm) / (float)C + a.eps);
  if (a.rstd && threadIdx.x % W::kLanes == 0) a.rstd[row] = rstd;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int run = run0 + W::kRuns * j;
    float w[8], y[8];
    if (a.w) load8<P, EIGHTS>((const P*)a.w, run * kRun, l16, C, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = v[j][e] * rstd;
      if (a.w) y[e] *= w[e];
      if (run * kRun + l16 * 8 + e >= C) y[e] = 0.f;   // also where the row's rstd is not finite
    }
    if (a.y) store8<T, EIGHTS>((T*)a.y + row * C, run * kRun + l16 * 8, 0, C, y);
    if (a.y8.codes) {
      uint32_t s;
      const uint2 c = encode8(y, s);
      if (run < runs) store_codes(a.y8.codes + (row * runs + run) * kRun, l16, c);
      if (WAVES > 0) {
        if (run < ss && l16 == 0) a.y8.scales[row * ss + run] = run < runs ? (uint8_t)s : 0;
      } else if (l16 == 0) {   // one run: the whole word of scales
        *(uint32_t*)(a.y8.scales + row * ss) = s;
      }
    }
  }
}

// Teams walk over the rows (the grid is a fixed number of workgroups), the next row on its way while one is worked on, and
// keep their part of dw in registers; the workgroup's sum goes to `part`, and param_sum_kernel (rows8.hip) adds those up in a
// fixed order: no atomics, the same result every time.
// Above 8192 channels, where a compute unit has room for one row's team and the next row's loads, 3.6 TB/s (bf16 3800 x 8960 75 us).
template <typename T, typename P, bool EIGHTS, int WAVES, int NV, bool DS>
__global__ __launch_bounds__(Team<WAVES>::kThreads, EIGHTS && WAVES < 16 ? 2 : 1) void rms_norm_grad_kernel(RmsGradArgs a) {
  using W = Team<WAVES>;
  __shared__ float sm[2][WAVES > 1 ? WAVES : 1];
  __shared__ float join[W::kTeams > 1 ? W::kTeams * W::kLanes * 8 : 1];
  const int l16 = threadIdx.x & 15, C = a.C;
  const int team = threadIdx.x / W::kLanes, lane = threadIdx.x % W::kLanes, run0 = lane >> 4;
  auto first = [&](int j) { return (run0 + W::kRuns * j) * kRun; };
  // the rows as they lie stay in registers, and are widened in each pass: a row's and the next one's are half, or a quarter, of the floats.
  // The widest rows take the weights from the cache for each row, and keep dw in LDS, where they pass what a lane of 16 waves has.
  constexpr bool kLean = WAVES == 16 && NV > 1, kAhead = DS && !(kLean && (sizeof(T) == 4 || !EIGHTS));
  __shared__ __attribute__((aligned(16))) f32x4 held[kLean ? 2 * NV * W::kThreads : 1];
  float w[NV][8], dw[NV][8];
  auto weights = [&](int j) {
    if (a.w) load8<P, EIGHTS>((const P*)a.w, first(j), l16, C, w[j]);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (!a.w) w[j][e] = 1.f;
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (!kLean) weights(j);
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[j][e] = 0.f;
    if constexpr (kLean) held[2 * j * W::kThreads + lane] = held[(2 * j + 1) * W::kThreads + lane] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  struct Row {
    float rstd;
    Raw8<T> dy[NV], s[NV], ds[DS ? NV : 1];
  };
  auto load_ds = [&](Row& x, int64_t row) {
#pragma unroll
    for (int j = 0; j < NV; ++j) x.ds[j] = load_part<T, EIGHTS>((const T*)a.ds + row * C, first(j), l16, C);
  };
  auto load = [&](Row& x, int64_t row) {
    x.rstd = a.rstd[row];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      x.dy[j] = load_part<T, EIGHTS>((const T*)a.dy + row * C, first(j), l16, C);
      x.s[j] = load_part<T, EIGHTS>((const T*)a.s + row * a.s_stride, first(j), l16, C);
    }
    if constexpr (kAhead) load_ds(x, row);
  };
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * W::kTeams;
  int64_t row = (int64_t)blockIdx.x * W::kTeams + team;
  Row next;
  if (row < a.rows) load(next, row);
  for (; row < a.rows; row += step, turn ^= 1) {
    Row x = next;
    if constexpr (DS && !kAhead) load_ds(x, row);
    if (row + step < a.rows) load(next, row + step);
    settle<T, EIGHTS>(x.dy[NV - 1], first(NV - 1), l16, C);
    settle<T, EIGHTS>(x.s[NV - 1], first(NV - 1), l16, C);
    if constexpr (DS) settle<T, EIGHTS>(x.ds[NV - 1], first(NV - 1), l16, C);
    // past the row's end (in the last vectors only) dy and s are 0, and n has to be 0 too where rstd is not finite
    auto normed = [&](int j, int e) {
      const float n = (float)x.s[j].v[e] * x.rstd;
      return j == NV - 1 && first(j) + l16 * 8 + (EIGHTS ? 0 : e) >= C ? 0.f : n;
    };
    float s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (kLean) {
        weights(j);
        *(f32x4*)&dw[j][0] = held[2 * j * W::kThreads + lane];
        *(f32x4*)&dw[j][4] = held[(2 * j + 1) * W::kThreads + lane];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float dy = (float)x.dy[j].v[e], n = normed(j, e);
        s2 = fmaf(dy * w[j][e], n, s2);
        dw[j][e] = fmaf(dy, n, dw[j][e]);
      }
      if constexpr (kLean) {
        held[2 * j * W::kThreads + lane] = *(const f32x4*)&dw[j][0];
        held[(2 * j + 1) * W::kThreads + lane] = *(const f32x4*)&dw[j][4];
      }
    }
    const float m2 = team_sum<WAVES>(s2, sm[turn]) / (float)C;
    if constexpr (kLean) asm volatile("" ::: "memory");   // the weights again, not kept from above
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if constexpr (kLean) weights(j);
      float dx[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dx[e] = x.rstd * ((float)x.dy[j].v[e] * w[j][e] - normed(j, e) * m2);
        if constexpr (DS) dx[e] += (float)x.ds[j].v[e];
      }
      store8<T, EIGHTS>((T*)a.dx + row * C, first(j) + l16 * 8, 0, C, dx);
    }
  }
  if (!a.part) return;
  float* const part = a.part + (int64_t)blockIdx.x * C;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if constexpr (W::kTeams > 1) {   // the teams hold the same channels: their sums meet in LDS
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 8; ++e) join[(team * 8 + e) * W::kLanes + lane] = dw[j][e];
      __syncthreads();
      for (int i = threadIdx.x; i < 8 * W::kLanes; i += W::kThreads) {   // element i / kLanes of lane i % kLanes
        float s = 0.f;
#pragma unroll
        for (int t = 0; t < W::kTeams; ++t) s += join[t * 8 * W::kLanes + i];
        const int l = i % W::kLanes, c = ((l >> 4) + W::kRuns * j) * kRun + (l & 15) * 8 + i / W::kLanes;
        if (c < C) part[c] = s;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (first(j) + l16 * 8 + e < C) part[first(j) + l16 * 8 + e] = kLean ? held[(2 * j + e / 4) * W::kThreads + lane][e % 4] : dw[j][e];
    }
  }
}

// ------------------------------------------------------------------------------------------------------------
// launches
// ------------------------------------------------------------------------------------------------------------
constexpr int kRmsGradBlocks = 512;   // two workgroups a CU: 768 took 51 us for 47.6 (17280 x 1536), and 140 for 116 (fp32 8000 x 4001)

// f(waves a row, vectors a lane): up to 4 vectors a lane up to WIDE channels, else 2. Fewer waves a row meet less; the gradient of fp32 rows
// and of those past 6144 channels has no registers for it (bf16 17280 x 1536, forward and back: 83.6 us with 3 vectors, 88.3 with 4 waves;
// 4000 x 8192, back: 73 with 4 vectors, 62 with 16 waves).
template <int WIDE, class F>
static int pick_rms_team(int C, F&& f) {
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  using I2 = std::integral_constant<int, 2>;
  using I3 = std::integral_constant<int, 3>;
  using I4 = std::integral_constant<int, 4>;
  using I16 = std::integral_constant<int, 16>;
  if (C <= 128) f(I0{}, I1{});
  else if (C <= 512) f(I1{}, I1{});
  else if (C <= 1024) f(I1{}, I2{});
  else if (C <= 2048) {
    if constexpr (WIDE == 0) f(I4{}, I1{});
    else if (C <= 1536) f(I1{}, I3{});
    else f(I1{}, I4{});
  } else if (C <= 4096) f(I4{}, I2{});
  else if (C <= 8192) {
    if constexpr (WIDE == 0) f(I16{}, I1{});
    else if (C <= 6144) f(I4{}, I3{});
    else if constexpr (WIDE == 8192) f(I4{}, I4{});
    else f(I16{}, I1{});
  } else f(I16{}, I2{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

// f(element type, parameter type, whether rows are read and written by whole vectors of 8)
template <class F>
static int pick_rms_types(int dtype, int param_dtype, int C, F&& f) {
  auto with = [&](auto t, auto p) { return C % 8 == 0 ? f(t, p, std::true_type{}) : f(t, p, std::false_type{}); };
  if (dtype == FVSR_DTYPE_BF16) return param_dtype == FVSR_DTYPE_BF16 ? with(bf16{}, bf16{}) : with(bf16{}, float{});
  return with(float{}, float{});   // fp32 tokens take fp32 parameters
}

int launch_rms_norm(int dtype, int param_dtype, const void* x, int64_t x_stride, const void* r, int64_t rows, int C, float eps,
                    const void* w, void* y, Out8 y8, void* s, float* rstd, hipStream_t stream) {
  if (rows <= 0) return FVSR_OK;
  const RmsArgs a{x, x_stride, r, rows, C, eps, w, y, y8, s, rstd};
  return pick_rms_types(dtype, param_dtype, C, [&](auto t, auto p, auto v) {
    return pick_rms_team<8192>(C, [&](auto waves, auto nv) {
      using W = Team<decltype(waves)::value>;
      hipLaunchKernelGGL((rms_norm_kernel<decltype(t), decltype(p), decltype(v)::value, decltype(waves)::value, decltype(nv)::value>),
                         dim3((unsigned)ceil_div(rows, W::kTeams)), dim3(W::kThreads), 0, stream, a);
    });
  });
}

// Workgroups of the gradient. One, for a few rows a team, has dw in it and needs no second launch. One and more, us of a graph's
// calls, and with the host's: 128 rows of 128 5.8, 10.1 and 5.1, 13.7; 32 of 512 5.9, 10.0 and 5.2, 14.0; 16 of 1000 5.6, 10.0 and 6.3,
// 13.9; 8 of 1536 5.1, 10.0 and 7.1, 14.2; 4 of 4096 7.4, 9.7 and 7.6, 13.8. Twice the rows lose: 64 of 512 9.6 and 5.4, 32 of 1000 9.3 and
// 6.6, 8 of 4096 11.1 and 7.6, 4 of 8960 13.5 and 12.2.
int64_t rms_grad_blocks(int64_t rows, int C) {
  if (rows <= (C <= 128 ? 128 : C <= 512 ? 32 : C <= 1024 ? 16 : C <= 2048 ? 8 : C <= 8192 ? 4 : 1)) return std::min<int64_t>(rows, 1);
  return std::min<int64_t>(kRmsGradBlocks, C <= 128 ? ceil_div(rows, 32) : C <= 2048 ? ceil_div(rows, 8) : ceil_div(rows, 2));
}

int launch_rms_norm_grad(int dtype, int param_dtype, const void* dy, const void* s, int64_t s_stride, const float* rstd,
                         const void* ds, int64_t rows, int C, const void* w, void* dx, float* dw, float* part,
                         hipStream_t stream) {
  const int64_t blocks = rms_grad_blocks(rows, C);
  if (blocks > 0) {
    const RmsGradArgs a{dy, s, s_stride, rstd, ds, rows, C, w, dx, !dw ? nullptr : blocks == 1 ? dw : part};
    const int rc = pick_rms_types(dtype, param_dtype, C, [&](auto t, auto p, auto v) {
      return pick_rms_team<sizeof(t) == 2 ? 6144 : 0>(C, [&](auto waves, auto nv) {
        constexpr int W = decltype(waves)::value, N = decltype(nv)::value;
        constexpr bool V = decltype(v)::value;
        const dim3 grid((unsigned)blocks), block(Team<W>::kThreads);
        if (ds) hipLaunchKernelGGL((rms_norm_grad_kernel<decltype(t), decltype(p), V, W, N, true>), grid, block, 0, stream, a);
        else hipLaunchKernelGGL((rms_norm_grad_kernel<decltype(t), decltype(p), V, W, N, false>), grid, block, 0, stream, a);
      });
    });
    if (rc) return rc;
  }
  return dw && blocks != 1 ? launch_param_sum(part, (int)blocks, C, C, dw, nullptr, stream) : FVSR_OK;
}

}  // namespace fvsr
