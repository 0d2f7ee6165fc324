// Rotary positions of several axes (time, height, width) for q and k in one launch, for gfx950 (MI355X).
//
// Pair i of a head, (a, b), belongs to one axis and turns by t = position on that axis * frequency[i]:
//   a' = a cos t - b sin t,  b' = a sin t + b cos t        (the gradient turns back: sin t changes its sign)
// Pairs are neighbours (channels 2 i, 2 i + 1) or halves (i, pairs + i); channels past the pairs are copied.
//
// Memory-bound: q and k move once. The angle is taken in 64 bits, in turns, and only what is left of its quarter in 32: a
// position of 10^5 keeps its angle to 10^-11, and the sine and cosine to their own last bits. A thread computes those of its
// pairs once and uses them for as many heads as it holds.
#include <algorithm>

#include "blocks8.hpp"

namespace fvsr {

struct RotaryPart {
  const void* x;
  void* out;
  int heads;
  int64_t xt, xh, ot, oh;   // elements between tokens and between heads
};

struct RotaryArgs {
  RotaryPart q, k;          // k.heads may be 0
  int64_t tokens;
  int D, pairs;
  const void* pos;          // (axes, tokens)
  int pos64;
  int end1, end2;           // pairs [0, end1) are of axis 0, [end1, end2) of axis 1, the others of axis 2
  const double* freq;       // (pairs)
  int back;                 // the gradient
  int units, span;          // units of kPairs pairs (then of 8 copied channels) a head; heads a thread
  int each;                 // tokens a workgroup
  uint32_t by_units;        // 2^16 / units, rounded up: a thread's number (below 256) times it, >> 16, is the quotient
};

// Sine and cosine of an angle in turns, by their series to x^9 and x^10 over an eighth of a turn to either side (off by less than
// 2^-29 there) and the quarter's symmetries.
__device__ __forceinline__ void sincos_turns(double turns, float& sine, float& cosine) {
  const double quarters = 4. * (turns - rint(turns)), whole = rint(quarters);
  const float x = (float)(quarters - whole) * 1.5707963267948966f, xx = x * x;
  const int q = (int)whole;
  float s = fmaf(xx, 1.f / 362880, -1.f / 5040), c = fmaf(xx, -1.f / 3628800, 1.f / 40320);
  s = fmaf(xx, s, 1.f / 120);
  c = fmaf(xx, c, -1.f / 720);
  s = fmaf(xx, s, -1.f / 6);
  c = fmaf(xx, c, 1.f / 24);
  s = fmaf(x * xx, s, x);
  c = fmaf(xx, c, -0.5f);
  c = fmaf(xx, c, 1.f);
  const float a = q & 1 ? c : s, b = q & 1 ? s : c;
  sine = q & 2 ? -a : a;
  cosine = (q + 1) & 2 ? -b : b;
}

// kPairs: 4 neighbours (16 bytes of bf16 a thread, adjacent threads adjacent) or 8 in halves (16 bytes of either)
template <typename T, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  constexpr int kPairs = HALVES ? 8 : 4;
  typedef T any_half __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  const int mine = (int)(threadIdx.x * a.by_units >> 16);
  const int64_t token = (int64_t)blockIdx.x * a.each + mine;
  if (mine >= a.each || token >= a.tokens) return;
  const int unit = (int)threadIdx.x - mine * a.units, first = unit * kPairs;
  const int heads = a.q.heads + a.k.heads, h0 = (int)blockIdx.y * a.span, h1 = min(heads, h0 + a.span);
  const T* const qx = (const T*)a.q.x + token * a.q.xt;
  const T* const kx = (const T*)a.k.x + token * a.k.xt;
  T* const qo = (T*)a.q.out + token * a.q.ot;
  T* const ko = (T*)a.k.out + token * a.k.ot;
  auto from = [&](int h) { return h < a.q.heads ? qx + h * a.q.xh : kx + (h - a.q.heads) * a.k.xh; };
  auto to = [&](int h) { return h < a.q.heads ? qo + h * a.q.oh : ko + (h - a.q.heads) * a.k.oh; };
  if (first >= a.pairs) {   // channels past the pairs: 8 a unit
    const int c0 = 2 * a.pairs + 8 * (unit - (a.pairs + kPairs - 1) / kPairs), n = min(8, a.D - c0);
    for (int h = h0; h < h1; ++h) {
      const T* x = from(h) + c0;
      T* o = to(h) + c0;
      if (x == o) continue;
      if (n == 8) {
        *(any_half*)o = *(const any_half*)x;
      } else {
        for (int e = 0; e < n; ++e) o[e] = x[e];
      }
    }
    return;
  }
  const int n = min(kPairs, a.pairs - first);
  constexpr int kAhead = sizeof(T) == 2 && !HALVES ? 8 : 4;   // heads whose loads are under way together
  any_half u[kAhead], v[kAhead];
  auto load = [&](int h) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (h + j < h1) {
        const T* x = from(h + j) + (HALVES ? first : 2 * first);
        u[j] = *(const any_half*)x;
        if constexpr (HALVES) v[j] = *(const any_half*)(x + a.pairs);
      }
    }
  };
  if (n == kPairs) load(h0);   // on their way while the angles are made
  float c[kPairs], s[kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) {
    const int p = min(first + e, a.pairs - 1), axis = p < a.end1 ? 0 : p < a.end2 ? 1 : 2;
    const int64_t at = axis * a.tokens + token;
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
    sincos_turns(pos * a.freq[p] * 0.15915494309189535, s[e], c[e]);   // 1 / (2 pi)
    if (a.back) s[e] = -s[e];
  }
  if (n == kPairs) {
    for (int h = h0; h < h1; h += kAhead) {
      any_half x[kAhead], y[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if constexpr (HALVES) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = (float)u[j][e], q = (float)v[j][e];
            x[j][e] = (T)(p * c[e] - q * s[e]);
            y[j][e] = (T)(p * s[e] + q * c[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float p = (float)u[j][2 * e], q = (float)u[j][2 * e + 1];
            x[j][2 * e] = (T)(p * c[e] - q * s[e]);
            x[j][2 * e + 1] = (T)(p * s[e] + q * c[e]);
          }
        }
      }
      load(h + kAhead);
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        if (h + j < h1) {
          T* o = to(h + j) + (HALVES ? first : 2 * first);
          *(any_half*)o = x[j];
          if constexpr (HALVES) *(any_half*)(o + a.pairs) = y[j];
        }
      }
    }
    return;
  }
  for (int h = h0; h < h1; ++h) {   // the last unit of a number of pairs that does not divide
    const T* x = from(h);
    T* o = to(h);
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      if (e < n) {
        const int i0 = HALVES ? first + e : 2 * (first + e), i1 = HALVES ? i0 + a.pairs : i0 + 1;
        const float p = (float)x[i0], q = (float)x[i1];
        o[i0] = (T)(p * c[e] - q * s[e]);
        o[i1] = (T)(p * s[e] + q * c[e]);
      }
    }
  }
}

int launch_rotary(int dtype, const fvsr_heads* q, const fvsr_heads* q_out, const fvsr_heads* k, const fvsr_heads* k_out,
                  int64_t tokens, int D, const void* pos, int pos64, const double* freq, int axes, const int32_t* axis_pairs,
                  int halves, int back, hipStream_t stream) {
  auto part = [](const fvsr_heads* x, const fvsr_heads* o) {
    return x ? RotaryPart{x->data, o->data, x->heads, x->token_stride, x->head_stride, o->token_stride, o->head_stride}
             : RotaryPart{};
  };
  RotaryArgs a{part(q, q_out), part(k, k_out), tokens, D, 0, pos, pos64, 0, 0, freq, back, 0, 0, 0, 0};
  for (int i = 0; i < axes; ++i) a.pairs += axis_pairs[i];
  a.end1 = axis_pairs[0];
  a.end2 = a.end1 + (axes > 1 ? axis_pairs[1] : 0);
  const int per = halves ? 8 : 4;
  a.units = (int)(ceil_div(a.pairs, per) + ceil_div(D - 2 * a.pairs, 8));
  a.each = 256 / a.units;
  a.by_units = 65536 / a.units + 1;
  const int heads = a.q.heads + a.k.heads;
  // heads a thread: as many as leave the card 2^18 threads, since each repeats the angles of its pairs
  const int64_t threads = tokens * a.units;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(std::min(heads, 65535), ((int64_t)1 << 18) / threads));
  a.span = (int)ceil_div(heads, parts);
  const int64_t blocks = ceil_div(tokens, a.each);
  if (blocks >= ((int64_t)1 << 24)) return set_error(FVSR_ERR_UNSUPPORTED, "too many tokens for one launch");
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(heads, a.span));
  auto go = [&](auto t) {
    using T = decltype(t);
    if (halves) hipLaunchKernelGGL((rotary_kernel<T, true>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<T, false>), grid, dim3(256), 0, stream, a);
  };
  if (dtype == FVSR_DTYPE_BF16) go(bf16{});
  else go(float{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

}  // namespace fvsr
