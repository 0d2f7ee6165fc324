// Rotary positions of several axes (time, height, width) for q and k in one launch, for gfx950 (MI355X).
//
// Pair i of a head, (a, b), belongs to one axis and turns by t = position on that axis * frequency[i]:
//   a' = a cos t - b sin t,  b' = a sin t + b cos t        (the gradient turns back: sin t changes its sign)
// Pairs are neighbours (channels 2 i, 2 i + 1) or halves (i, pairs + i); channels past the pairs are copied.
//
// Memory-bound: q and k move once. The angle is taken in 64 bits, in turns, and only what is left of its quarter in 32: a
// position of 10^5 keeps its angle to 10^-11, and the sine and cosine to their own last bits. A thread computes those of its
// pairs once and uses them for as many heads as it holds.
//
// bf16 17280 tokens, 12 + 12 heads of 128: 47.6 us, 4.5 TB/s (a copy: 4.7), with the operands in the memory-side cache 33.8; in halves 51.
// 4001 tokens of 9 + 3 heads of 80 in fp32: 11.2, a launch, the chain from a position to its sine, and 31 MB.
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
  int units, span;          // units of a head; heads a thread
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

// The first `by` of 8 values taken out, the others moved to the front.
template <typename T, typename V>
__device__ __forceinline__ V moved(V v, int by) {
  if constexpr (sizeof(T) == 2) {
    u32x4 x = __builtin_bit_cast(u32x4, v);
    if (by & 4) x = u32x4{x[2], x[3], 0, 0};
    if (by & 2) x = u32x4{x[1], x[2], x[3], 0};
    if (by & 1) x = u32x4{x[0] >> 16 | x[1] << 16, x[1] >> 16 | x[2] << 16, x[2] >> 16 | x[3] << 16, x[3] >> 16};
    return __builtin_bit_cast(V, x);
  } else {
#pragma unroll
    for (int b = 4; b > 0; b >>= 1)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = !(by & b) ? v[e] : e + b < 8 ? v[e + b] : 0;
    return v;
  }
}

// A thread's unit is 8 channels of neighbouring pairs (kPairs 4, the last of them perhaps past the pairs, and copied), or 8 channels
// of either half (kPairs 8), or, behind the halves, 8 channels that are copied. All are read by whole vectors, several heads at once,
// those that would pass the head's end from 8 before it: a unit that went channel by channel, head after head, would be what the
// others wait for (17280 tokens, 20 heads of 80 channels, 33 pairs: 78 us so, 31 now).
// WHOLE: units of whole vectors only, either turned or copied.
template <typename T, bool HALVES, bool WHOLE>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  constexpr int kPairs = HALVES ? 8 : 4;
  typedef T any_half __attribute__((ext_vector_type(8), aligned(sizeof(T))));
  typedef T half8 __attribute__((ext_vector_type(8)));
  const int mine = (int)(threadIdx.x * a.by_units >> 16);
  const int64_t token = (int64_t)blockIdx.x * a.each + mine;
  if (mine >= a.each || token >= a.tokens) return;
  const int unit = (int)threadIdx.x - mine * a.units, first = unit * kPairs, D = a.D;
  const int heads = a.q.heads + a.k.heads, h0 = (int)blockIdx.y * a.span, h1 = min(heads, h0 + a.span);
  const T* const qx = (const T*)a.q.x + token * a.q.xt;
  const T* const kx = (const T*)a.k.x + token * a.k.xt;
  T* const qo = (T*)a.q.out + token * a.q.ot;
  T* const ko = (T*)a.k.out + token * a.k.ot;
  auto from = [&](int h) { return h < a.q.heads ? qx + h * a.q.xh : kx + (h - a.q.heads) * a.k.xh; };
  auto to = [&](int h) { return h < a.q.heads ? qo + h * a.q.oh : ko + (h - a.q.heads) * a.k.oh; };
  // pairs that turn, first channel, channels (of either half); the first channel of the other half
  const int turned = max(0, min(kPairs, a.pairs - first)), n = WHOLE ? kPairs : turned;
  const int beyond = unit - (a.pairs + kPairs - 1) / kPairs;
  const int c0 = !HALVES ? 2 * first : turned > 0 ? first : 2 * a.pairs + 8 * beyond;
  const int count = WHOLE ? 8 : HALVES && n > 0 ? n : min(8, D - c0);
  const int d0 = a.pairs + first;
  constexpr int kAhead = sizeof(T) == 2 && !HALVES ? 8 : 4;   // heads whose loads are under way together
  half8 u[kAhead], v[kAhead];
  if (WHOLE && turned == 0) {
    for (int h = h0; h < h1; ++h)
      if (to(h) != from(h)) *(any_half*)(to(h) + c0) = *(const any_half*)(from(h) + c0);
    return;
  }
  const int at0 = WHOLE ? c0 : max(0, min(c0, D - 8)), at1 = WHOLE ? d0 : max(0, min(d0, D - 8));
  auto fetch = [&](const T* x, int at) {
    half8 r;
    if (WHOLE || D >= 8) {
      r = *(const any_half*)(x + at);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = e < D ? x[e] : (T)0.f;
    }
    return r;
  };
  auto load = [&](int h) {
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (h + j < h1) {
        u[j] = fetch(from(h + j), at0);
        if constexpr (HALVES)
          if (n > 0) v[j] = fetch(from(h + j), at1);
      }
    }
  };
  load(h0);   // on their way while the angles are made
  float c[kPairs], s[kPairs];
#pragma unroll
  for (int e = 0; e < kPairs; ++e) {
    c[e] = s[e] = 0.f;
    if (e >= n) continue;   // WHOLE: all or none
    const int p = first + e, axis = p < a.end1 ? 0 : p < a.end2 ? 1 : 2;
    const int64_t at = axis * a.tokens + token;
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at] : (double)((const int32_t*)a.pos)[at];
    sincos_turns(pos * a.freq[p] * 0.15915494309189535, s[e], c[e]);   // 1 / (2 pi)
    if (a.back) s[e] = -s[e];
  }
  auto store = [&](T* o, half8 x) {
    if (count == 8) {
      *(any_half*)o = x;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < count) o[e] = x[e];
    }
  };
  for (int h = h0; h < h1; h += kAhead) {
    half8 x[kAhead], y[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      x[j] = WHOLE || at0 == c0 ? u[j] : moved<T>(u[j], c0 - at0);
      if constexpr (HALVES) {
        y[j] = WHOLE || at1 == d0 ? v[j] : moved<T>(v[j], d0 - at1);
        if (n > 0) {   // past n: not stored
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = (float)x[j][e], q = (float)y[j][e];
            x[j][e] = (T)(p * c[e] - q * s[e]);
            y[j][e] = (T)(p * s[e] + q * c[e]);
          }
        }
      } else if (n > 0) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = (float)x[j][2 * e], q = (float)x[j][2 * e + 1];
          const T p2 = (T)(p * c[e] - q * s[e]), q2 = (T)(p * s[e] + q * c[e]);
          x[j][2 * e] = WHOLE || e < n ? p2 : x[j][2 * e];
          x[j][2 * e + 1] = WHOLE || e < n ? q2 : x[j][2 * e + 1];
        }
      }
    }
    load(h + kAhead);
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      if (h + j < h1) {
        T* const o = to(h + j);
        if (n > 0 || o != from(h + j)) store(o + c0, x[j]);
        if constexpr (HALVES)
          if (n > 0) store(o + d0, y[j]);
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
  a.units = (int)(halves ? ceil_div(a.pairs, 8) + ceil_div(D - 2 * a.pairs, 8) : ceil_div(D, 8));
  a.each = 256 / a.units;
  a.by_units = 65536 / a.units + 1;
  const int heads = a.q.heads + a.k.heads;
  // Heads a thread: as many as leave the card 2^18 threads, since each repeats the angles of its pairs. 2000 and 8000 tokens of 24 heads,
  // 4000 of 40 in halves, us: 7.2, 17.0, 16.9; with 2^16 threads 7.1, 17.3, 19.7; 2^17 6.4, 17.3, 17.7; 2^19 8.9, 20.9, 19.4; 2^20 11.9,
  // 25.6, 21.7.
  const int64_t threads = tokens * a.units;
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(std::min(heads, 65535), ((int64_t)1 << 18) / threads));
  a.span = (int)ceil_div(heads, parts);
  const int64_t blocks = ceil_div(tokens, a.each);
  if (blocks >= ((int64_t)1 << 24)) return set_error(FVSR_ERR_UNSUPPORTED, "too many tokens for one launch");
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(heads, a.span));
  auto go = [&](auto t) {
    using T = decltype(t);
    const bool whole = a.pairs % (halves ? 8 : 4) == 0 && D % 8 == 0;
    auto with = [&](auto h) {
      constexpr bool H = decltype(h)::value;
      if (whole) hipLaunchKernelGGL((rotary_kernel<T, H, true>), grid, dim3(256), 0, stream, a);
      else hipLaunchKernelGGL((rotary_kernel<T, H, false>), grid, dim3(256), 0, stream, a);
    };
    if (halves) with(std::true_type{});
    else with(std::false_type{});
  };
  if (dtype == FVSR_DTYPE_BF16) go(bf16{});
  else go(float{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

}  // namespace fvsr
