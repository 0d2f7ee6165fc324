// Attention over packed sequences for gfx950 (MI355X), causal or whole, query heads in groups that share a key and value
// head, with its gradient.
//
//   S = scale Q K^T,  P = softmax(S) over the keys that a query sees,  O = P V,  lse = log(sum exp(S))
//   delta = sum over channels of dO O,  dP = dO V^T,  dS = P (dP - delta)
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO          (dK and dV summed over the group's query heads)
//
// Sequence b has queries cu_q[b] .. cu_q[b + 1] - 1 and keys from cu_k[b] on. Query i of m sees all n keys, or, causal, the
// first i + 1 + n - m. The lengths are on the device only: a workgroup finds its sequence from its number (block_of), and the grid is known
// from the totals.
//
// bf16 operands, fp32 sums on v_mfma_f32_32x32x16_bf16: S^T = K Q^T, so a lane owns a query, P packed to bf16 goes
// straight back in as the operand of O^T += V^T P^T, V^T read transposed from row-major LDS (ds_read_b64_tr_b16). P and dS are
// rounded to bf16 for those products (off by at most 2^-8 of themselves each); sums of P, the softmax and delta stay fp32.
//
// Figures below are of 12 heads of 128 over 17280 x 17280 rows, whole, unless said otherwise; a bf16 library product of 16384^3 reaches
// 1345 TFLOP/s on the same card.
#include <algorithm>

#include "attn_tile.hpp"
#include "packed_attn.hpp"
#include "teams.hpp"

namespace fvsr {
namespace {

constexpr int kRows = 128;      // rows of a block: 4 waves of 32
constexpr int kTile = 32;       // rows of a tile of the other side
constexpr float kRise = 4096.f, kAbove = 20.f, kAbove2 = 1048576.f;   // kAbove2 = 2^kAbove
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// A tile of 32 rows of HD channels in LDS (D <= HD, zeros past D): rows of 2 HD bytes, whose 16-byte chunks are XOR-swizzled by
// row so that both reads of a tile spread over all banks: 16 rows of one chunk (ds_read_b128), and 4 neighbouring rows (a
// multiple of 4 first) of 4 adjacent chunks (ds_read_b64_tr_b16).
template <int HD>
struct Tile {
  static constexpr int kRow = 2 * HD, kBytes = kTile * kRow, kChunks = HD / 8;
  static constexpr int kCopies = kBytes / 1024, kCopyRows = 1024 / kRow;   // a copy: 64 lanes of 16 bytes
  static constexpr int kT = HD / 16, kD = HD / 32;                         // products over the channels, blocks of channels
  static __device__ __forceinline__ int swz(int r) {
    return HD == 128 ? ((r & 3) << 2 | (r >> 2 & 3)) : ((r >> 1 & 1) << 2 | (r >> 2 & 3));
  }
};

// byte offset, for copy p of a tile, of the lane's chunk in rows `stride` bytes apart; past every buffer where the channels
// are past D
template <int HD>
__device__ __forceinline__ int copy_off(int p, int lane, int stride, int D) {
  using T = Tile<HD>;
  const int r = p * T::kCopyRows + lane / T::kChunks, chunk = lane % T::kChunks ^ T::swz(r);
  return chunk * 8 < D ? r * stride + chunk * 16 : (int)0x80000000;
}

// The buffer of rows row0 .. of a head whose rows end at `end`: what is past it reads as zeros. The base is 64 bits wide, so
// offsets of long caches do not wrap; 32 rows stay below 2^31 bytes.
__device__ __forceinline__ u32x4 rows_rsrc(const bf16* base, int64_t stride, int row0, int end, int D) {
  const int left = min(end - row0, kTile);
  const uint64_t at = (uint64_t)(base + (int64_t)row0 * stride);
  const uint32_t bytes = left <= 0 ? 0 : (uint32_t)((left - 1) * (int)stride + D) * 2;
  return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)at),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu)),
               (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

// the compiler moves no memory access across it
__device__ __forceinline__ void fence() { asm volatile("" ::: "memory"); }

// The loads so far have landed. Before a loop whose copies (which the compiler does not count) are waited for by their number: it
// would wait for none to be under way, every time round, where a load from before the loop might be.
__device__ __forceinline__ void loaded() {
  fence();
  FVSR_WAIT_VM_LGKM0(0);
  fence();
}

// The copies but the last `under_way` of this wave have landed, and every wave is past its reads.
template <int UNDER_WAY>
__device__ __forceinline__ void wait_and_sync_but(bool all) {
  fence();
  if (all) FVSR_WAIT_VM_LGKM0(0);
  else FVSR_WAIT_VM_LGKM0(UNDER_WAY);
  __builtin_amdgcn_s_barrier();
  fence();
}

// LDS offsets of a lane's operands within a tile. The swizzle being an XOR, an operand further on in the channels is the first
// one's offset XOR a constant, made where it is used: two registers instead of 16.
template <int HD>
struct Lanes {
  uint32_t row0, tr0;
  __device__ __forceinline__ Lanes() {
    using T = Tile<HD>;
    const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, G = lane >> 4, mm = lane & 15;
    row0 = l32 * T::kRow + (g ^ T::swz(l32)) * 16;
    const int r = 4 * (G >> 1) + (mm >> 2);
    tr0 = r * T::kRow + ((2 * (G & 1) + (mm >> 1 & 1)) ^ T::swz(r)) * 16 + (mm & 1) * 8;
  }
  // not known to be what it was: computed where it is used, and kept in no register across a loop
  __device__ __forceinline__ void again() { asm volatile("" : "+v"(row0), "+v"(tr0)); }
  // A operand of (tile rows) x (channels): row lane % 32, channels 16 t + 8 (lane / 32) ..
  __device__ __forceinline__ uint32_t row(int t) const { return row0 ^ (uint32_t)(32 * t); }
  // A operand of (channels) x (tile rows), transposed: channels 32 d .., rows 16 u + 8 ab + ..; 8 rows on, the swizzle's bit 1 turns
  __device__ __forceinline__ uint32_t tr(int ab, int u, int d) const {
    return (tr0 ^ (uint32_t)(64 * d + 32 * ab)) + (uint32_t)((16 * u + 8 * ab) * Tile<HD>::kRow);
  }
};

// (32 tile rows) x (32 columns, one a lane pair): the tile's rows times the lane's row b. Element i of the result is tile row
// 8 (i / 4) + 4 (lane / 32) + i % 4.
template <int HD>
__device__ __forceinline__ f32x16 rows_times(lds_char* tile, const Lanes<HD>& at, const bf16x8 (&b)[Tile<HD>::kT],
                                             f32x16 s = f32x16{}) {
#pragma unroll
  for (int t = 0; t < Tile<HD>::kT; ++t)
    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const lds_bf16x8*)(tile + at.row(t)), b[t], s, 0, 0, 0);
  return s;
}

// acc (channels x columns) += tile^T w, w packed from elements laid out as above
template <int HD>
__device__ __forceinline__ void add_packed(lds_char* tile, const Lanes<HD>& at, const bf16x8 (&w)[2], f32x16 (&acc)[Tile<HD>::kD]) {
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int d = 0; d < Tile<HD>::kD; ++d) {
      const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + at.tr(0, u, d)));
      const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(tile + at.tr(1, u, d)));
      // whole-vector concatenation: element-wise assembly of the operand is mis-lowered (one dword duplicated)
      const bf16x8 a = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
      acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, w[u], acc[d], 0, 0, 0);
    }
}

// whether a tile holds an infinity or NaN
template <int HD>
__device__ __forceinline__ bool any_odd(lds_char* tile) {
  uint32_t most = 0;
#pragma unroll
  for (int i = 0; i < Tile<HD>::kBytes / 1024; ++i) {
    const u32x4 x = *(const lds_u32x4*)(tile + i * 1024 + (threadIdx.x & 63) * 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) most |= (x[e] & 0x7f807f80u) + 0x00800080u;   // an exponent of all ones carries into the sign's place
  }
  return __ballot((most & 0x80008000u) != 0) != 0;
}

// The same one tile row after another, without those that the lane's column does not see: 0 times an infinity or NaN there
// would be NaN. `seen`: a bit a tile row. Slow, and reached only where a tile that is not seen whole holds such a value.
template <int HD>
__device__ __forceinline__ void add_seen(lds_char* tile, const f32x16& w, uint32_t seen, f32x16 (&acc)[Tile<HD>::kD]) {
  using T = Tile<HD>;
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll 1
  for (int r = 0; r < kTile; ++r) {
    const int i = (r >> 3) * 4 + (r & 3);
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) x = e == i ? w[e] : x;
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    const float p = __uint_as_float((r >> 2 & 1) ? both[1] : both[0]);   // held by the half of lanes that owns row r
    const bool see = seen >> r & 1;
#pragma unroll
    for (int d = 0; d < T::kD; ++d) {
      __builtin_amdgcn_sched_barrier(0);   // a few registers at a time: not to spill for what is rare
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int chunk = 4 * d + c;   // channels 32 d + 8 c + 4 g ..
        const bf16x4 v = *(const __attribute__((address_space(3))) bf16x4*)(tile + r * T::kRow + (chunk ^ T::swz(r)) * 16 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[d][4 * c + e] = see ? fmaf(p, (float)v[e], acc[d][4 * c + e]) : acc[d][4 * c + e];
      }
    }
  }
}

// bits lo .. hi - 1
__device__ __forceinline__ uint32_t bits(int lo, int hi) {
  const uint32_t below = hi >= 32 ? ~0u : (1u << max(hi, 0)) - 1, from = lo >= 32 ? 0u : ~0u << max(lo, 0);
  return below & from;
}

// the tile row of element i of a product, but for 4 (lane / 32)
constexpr int elem_row(int i) { return 8 * (i >> 2) + (i & 3); }

__device__ __forceinline__ void pack(const f32x16& p, bf16x8 (&w)[2]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = (bf16)p[i];
}

// acc += tile^T w, of which, MASKED, the lane's column sees tile rows lo .. hi - 1 (w is 0 in the others); `whole`: all of the wave's see
// all; `fine`: what rounding w to bf16 leaves is added too
template <int HD, bool MASKED>
__device__ __forceinline__ void add_times(lds_char* tile, const Lanes<HD>& at, const f32x16& w, int lo, int hi, bool whole, bool fine,
                                          f32x16 (&acc)[Tile<HD>::kD]) {
  if (MASKED && !whole && any_odd<HD>(tile)) return add_seen<HD>(tile, w, bits(lo, hi), acc);
  bf16x8 p[2];
  pack(w, p);
  add_packed<HD>(tile, at, p, acc);
  if (MASKED && fine) {
    f32x16 left;
#pragma unroll
    for (int i = 0; i < 16; ++i) left[i] = w[i] - (float)p[i >> 3][i & 7];
    pack(left, p);
    add_packed<HD>(tile, at, p, acc);
  }
}

// the lane's row (channels 16 t + 8 (lane / 32) .. of it) as the other operand; zeros where there is none
template <int HD>
__device__ __forceinline__ void load_row(const bf16* row, bool there, int D, bf16x8 (&b)[Tile<HD>::kT]) {
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int t = 0; t < Tile<HD>::kT; ++t) {
    b[t] = bf16x8{};
    if (there && 16 * t + 8 * g < D) b[t] = *(const bf16x8*)(row + 16 * t + 8 * g);
  }
}

// and back: acc (channels x columns) times `by` into the lane's row
template <int HD>
__device__ __forceinline__ void store_row(bf16* row, int D, const f32x16 (&acc)[Tile<HD>::kD], float by) {
  const int g = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int d = 0; d < Tile<HD>::kD; ++d)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int ch = 32 * d + 8 * c;
      bf16x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = (bf16)(acc[d][4 * c + e] * by);
      if (ch < D) *(bf16x4*)(row + ch + 4 * g) = x;
    }
}

// ---- sequences ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int within(int x, int lo, int hi) { return min(max(x, lo), hi); }

// Rows of a sequence, whatever the offsets hold: inside the tensors.
struct Span {
  int q0, nq, k0, nk, room;   // room: keys up to the next sequence's, nk of them in use
};
__device__ __forceinline__ Span span_from(const PackedArgs& a, int q0, int q1, int k0, int k1, int used) {
  Span s;
  s.q0 = within(q0, 0, a.tq);
  s.nq = within(q1, s.q0, a.tq) - s.q0;
  s.k0 = within(k0, 0, a.tk);
  s.room = within(k1, s.k0, a.tk) - s.k0;
  s.nk = a.used_k ? within(used, 0, s.room) : s.room;
  return s;
}
__device__ __forceinline__ Span span_of(const PackedArgs& a, int b) {
  return span_from(a, uniform(a.cu_q[b]), uniform(a.cu_q[b + 1]), uniform(a.cu_k[b]), uniform(a.cu_k[b + 1]),
                   a.used_k ? uniform(a.used_k[b]) : 0);
}

// A block of kRows rows: of sequence b, from its row `row` on (b below 0, or not below the sequences: of none). Rows of no sequence,
// which are cleared where the call asks for it: [lo, hi), or of those below `lo` and from `hi` on every `step`-th kRows, from chunk `at`.
struct Block {
  int b, row;
  int lo, hi, at, step;
};
template <class F>
__device__ __forceinline__ void for_outside(const Block& x, int total, F&& f) {
  if (x.step == 0) {
    if (x.hi > x.lo) f(x.lo, x.hi);
    return;
  }
  const int lead = (x.lo + kRows - 1) / kRows, tail = (total - x.hi + kRows - 1) / kRows;
  for (int c = x.at; c < lead + tail; c += x.step) {
    const int from = c < lead ? c * kRows : x.hi + (c - lead) * kRows;
    f(from, min(from + kRows, c < lead ? x.lo : total));
  }
}

// Workgroup n's block, and the sequence's span; blocks of queries in falling order, since a sequence's last rows see most where it is
// causal. Offsets of up to 63 sequences are held by the lanes of a wave, which look for theirs side by side: one round trip to memory,
// where the blocks of short sequences spend much of their time.
//
// Blocks of sequence b begin in slot first row / kRows + b, so that slots never collide, or, short sequences, one behind another: then the
// lanes count their blocks first. Workgroups without work among the others leave two on one compute unit and none on the next, which
// costs the more the shorter the sequences: forward and gradient of 12 heads of 128, us, dense and with gaps: 40 sequences of 128 15.5, 61
// and 21.5, 87; 32 of 512 67, 241 and 71, 260; 5 of 512 15.8 and 20.7 (forward); but 40 causal ones of 1024 206, 694 and 200, 667. From 64
// sequences on, which the lanes do not hold, all have gaps: dense blocks of so many are not built, and not measured.
template <bool KEYS>   // blocks of keys, or of queries
__device__ __forceinline__ Block block_of(const PackedArgs& a, int n, Span& span) {
  const int lane = threadIdx.x & 63, seqs = a.seqs, total = KEYS ? a.tk : a.tq, slots = total / kRows + seqs + 1;
  const int at = min(lane, seqs);
  const int q = a.cu_q[at], k = a.cu_k[at], used = a.used_k ? a.used_k[min(lane, seqs - 1)] : 0;
  Block x{-1, 0, 0, 0, 0, 0};
  auto of = [](int v, int l) { return __builtin_amdgcn_readlane(v, l); };
  if (seqs < 64 && total <= 4 * kRows * seqs) {
    const int mine = KEYS ? k : q, next = __shfl_down(mine, 1), from = within(mine, 0, total);   // by every lane
    const int rows = lane < seqs ? within(next, from, total) - from : 0;
    const int blocks = (rows + kRows - 1) / kRows, upto = wave_scan_dpp(blocks);
    const int all = of(upto, 63), slot = KEYS ? n : all - 1 - n;
    if (n < all) {
      x.b = uniform(__popcll(__ballot(upto <= slot)));   // < seqs: the last lane's is all
      x.row = (slot - (of(upto, x.b) - of(blocks, x.b))) * kRows;
      span = span_from(a, of(q, x.b), of(q, x.b + 1), of(k, x.b), of(k, x.b + 1), of(used, x.b));
    } else {
      x.lo = of(from, 0);
      x.hi = within(of(mine, seqs), x.lo, total);
      x.at = n - all;
      x.step = max(1, slots - all);
    }
    return x;
  }
  const int32_t* const cu = KEYS ? a.cu_k : a.cu_q;
  const int slot = KEYS ? n : slots - 1 - n;
  int before = __popcll(__ballot(lane <= seqs && within(KEYS ? k : q, 0, total) / kRows + lane <= slot));
  for (int i = 64; i <= seqs; i += 64) {
    const bool is = i + lane <= seqs && within(cu[min(i + lane, seqs)], 0, total) / kRows + i + lane <= slot;
    before += __popcll(__ballot(is));
  }
  x.b = uniform(before) - 1;
  const int b = max(x.b, 0);   // <= seqs
  int first;                   // row of the sequence, or behind the last one
  if (seqs < 64) {
    first = within(of(KEYS ? k : q, b), 0, total);
    span = span_from(a, of(q, b), of(q, b + 1), of(k, b), of(k, b + 1), of(used, b));   // of no use where b is seqs
  } else {
    first = within(uniform(cu[b]), 0, total);
    span = span_of(a, min(b, seqs - 1));
  }
  x.row = x.b < 0 ? 0 : (slot - (first / kRows + x.b)) * kRows;
  if (x.b < 0) {
    x.lo = slot * kRows;
    x.hi = min(x.lo + kRows, first);
  } else if (x.b == seqs) {
    x.lo = min(first + max(x.row, 0), total);
    x.hi = min(x.lo + kRows, total);
  } else if (x.b == 0 && x.row == 0) {   // the rest of the rows before the first sequence
    x.lo = first / kRows * kRows;
    x.hi = first;
  }
  if (x.row < 0) x.b = seqs;   // offsets that fall: nothing here
  return x;
}

__device__ __forceinline__ void clear_rows(HeadView<bf16> o, int head, int lo, int hi, int D) {
  for (int e = threadIdx.x; e < (hi - lo) * (D / 8); e += blockDim.x)
    *(u32x4*)(o.p + (int64_t)(lo + e / (D / 8)) * o.t + head * o.h + e % (D / 8) * 8) = u32x4{0, 0, 0, 0};
}

// the keys that query i of a sequence sees (rows past the last query: as many as that one)
__device__ __forceinline__ int keys_seen(const PackedArgs& a, const Span& s, int i) {
  return a.causal ? within(min(i, s.nq - 1) + 1 + s.nk - s.nq, 0, s.nk) : s.nk;
}

// ---- forward -----------------------------------------------------------------------------------------------------------
// lse of a row from its reference and sum; kAbove is taken off both, for the logarithm to keep its last bits
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m - kAbove + __builtin_amdgcn_logf(l * kAbove2)) * kLn2;
}

// A softmax in progress for the lane's query: reference m (log2 units), sum l of this lane's half of the keys, unnormalised
// output (channels x queries).
template <int HD>
struct Soft {
  float m, l;
  f32x16 acc[Tile<HD>::kD];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < Tile<HD>::kD; ++d) acc[d] = f32x16{};
  }
  // a tile of keys k0 .. k0 + 31, of which, MASKED, the lane's query sees those below `lim`, and every one of the wave those below `all`
  template <bool MASKED>
  __device__ __forceinline__ void tile(lds_char* kt, lds_char* vt, Lanes<HD>& at, const bf16x8 (&q)[Tile<HD>::kT], int k0, int lim, int all,
                                       float c) {
    const int g = (threadIdx.x & 63) >> 5;
    f32x16 s = rows_times<HD>(kt, at, q);
    if (MASKED) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = elem_row(i) < lim - k0 - 4 * g ? s[i] : -INFINITY;
    }
    // The reference is kAbove more than the row's maximum in the first tile that it sees. Later ones are taken as they come while their
    // exponentials' sum stays below kRise (a bfloat16 P and a 32-bit sum are as near whatever the reference is); where it does not, or is
    // NaN, the reference rises to kAbove more than their maximum: rare, as it takes scores 32 above the first ones, and a branch of the whole
    // wave. The sums on the way stay below 2^8 n |V| over n keys, finite for every |V| below 2^120 / n; a row's largest term is 2^-20 |V| or
    // more, which fp32 holds to bfloat16's precision for values from 2^-120 on. With the maximum itself as the reference, rising at 2^8 took
    // 29 % where scores have a deviation of 8 (4096 x 4096, 12 heads of 64: 74 -> 95 us, 74 so), and rising at 2^32 values from 2^100 / n
    // on passed the largest float.
    float part = 0.f;
    f32x16 p;
    auto take = [&] {
      const float ref = m == -INFINITY ? 0.f : m;   // nothing seen yet
      part = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(s[i], c, -ref));
        part += p[i];
      }
    };
    bool rise = true;
    if (__ballot(m == -INFINITY) == 0) {
      take();
      rise = !(part <= kRise);
    }
    if (__ballot(rise) != 0) {
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      const float to = fmaxf(m, fmaf(pair_max(mx), c, kAbove));
      const float by = __builtin_amdgcn_exp2f(m - (to == -INFINITY ? 0.f : to));
      m = to;
      l *= by;
#pragma unroll
      for (int d = 0; d < Tile<HD>::kD; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] *= by;
      take();
    }
    s = p;
    l += part;
    add_times<HD, MASKED>(vt, at, s, 0, lim - k0, k0 + kTile <= all, false, acc);
  }
};

// The walk over tiles that every row sees whole, four a turn: a step makes S of tile T + 1, P of tile T and adds P V of tile T - 1,
// a product of the matrix core at a time with a share of the rest behind it, fenced so that this is the order they are issued in:
// the exponentials, the reads of operands four rounds ahead, and the copies of K(T + 4) and V(T + 2) run while the matrix core
// does. K and V have a ring of four tiles each: K(T) is read a step before, and V(T) a step after, P(T) is made.
//
// Bound by the matrix core (64 % of the card's cycles; 16 products of 32 cycles a tile and wave, two waves a SIMD) at the clock that such
// work leaves, 1.6 GHz: 1.60 ms, 1.15 PFLOP/s. Without the pipeline, one tile's S, P and P V after another: 1.88 ms; the rows' maximum in
// every tile instead of Soft's reference: 2.46 ms. 4 waves of 32 queries share the tiles, since a wave of 64 has no registers
// left for the next S beside its sums. Of 64 channels there are half the products for as many exponentials: 0.96 PFLOP/s. Causal, 783 us.
// 32 sequences of 512 read and write 201 MB in 66 us, 3.0 TB/s. The tiles behind the walk have one form, masked: with a second for whole
// ones the sums were in registers twice, and what that spilled was reloaded behind the copies under way (40 causal sequences of 1024 228 us,
// 199 now; of 512 90 and 74).
template <int HD>
__global__ __launch_bounds__(256, 2) void packed_forward_kernel(PackedArgs a) {
  using T = Tile<HD>;
  __shared__ __attribute__((aligned(1024))) char smem[8 * T::kBytes];   // [K, V][tile % 4]
  constexpr int kRing = 4 * T::kBytes;
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, wave = uniform(threadIdx.x >> 6);
  const int head = blockIdx.x % a.heads;
  Span s;
  const Block blk = block_of<false>(a, blockIdx.x / a.heads, s);
  if (a.clear)
    for_outside(blk, a.tq, [&](int lo, int hi) {
      if (a.clear & 1) clear_rows(a.o, head, lo, hi, a.D);
      if (a.lse)
        for (int r = lo + (int)threadIdx.x; r < hi; r += 256) a.lse[(int64_t)head * a.tq + r] = -INFINITY;
    });
  if (blk.b < 0 || blk.b >= a.seqs) return;
  if (blk.row >= s.nq) return;
  const int i = blk.row + wave * 32 + l32, lim = keys_seen(a, s, i);
  const int lim_min = keys_seen(a, s, blk.row + wave * 32), lim_max = keys_seen(a, s, blk.row + wave * 32 + 31);
  // tiles that some row of the block sees, and that every one sees all of
  const int tiles = (keys_seen(a, s, blk.row + kRows - 1) + kTile - 1) / kTile, full = keys_seen(a, s, blk.row) / kTile;

  const bf16* const kb = a.k.p + (int64_t)s.k0 * a.k.t + head / a.group * a.k.h;
  const bf16* const vb = a.v.p + (int64_t)s.k0 * a.v.t + head / a.group * a.v.h;
  constexpr int kMine = T::kCopies / 4;   // copies of a tile a wave makes
  int koff[kMine], voff[kMine];
#pragma unroll
  for (int p = 0; p < kMine; ++p) {
    koff[p] = copy_off<HD>(wave * kMine + p, lane, (int)a.k.t * 2, a.D);
    voff[p] = copy_off<HD>(wave * kMine + p, lane, (int)a.v.t * 2, a.D);
  }
  const uint32_t base = lds_addr(smem), mine = base + wave * kMine * 1024;
  lds_char* const lds = (lds_char*)(uintptr_t)base;
  // past the last tile, and before the first: zeros
  auto k_rsrc = [&](int t) { return rows_rsrc(kb, a.k.t, t * kTile, t < 0 ? t * kTile : s.nk, a.D); };
  auto v_rsrc = [&](int t) { return rows_rsrc(vb, a.v.t, t * kTile, t < 0 ? t * kTile : s.nk, a.D); };
  auto copy_k = [&](const u32x4& r, auto p, int slot) {
    dma16<decltype(p)::value * 1024>(r, mine + slot * T::kBytes, koff[decltype(p)::value], 0);
  };
  auto copy_v = [&](const u32x4& r, auto p, int slot) {
    dma16<kRing + decltype(p)::value * 1024>(r, mine + slot * T::kBytes, voff[decltype(p)::value], 0);
  };
  auto request = [&](int tk, int tv) {
    const u32x4 kr = k_rsrc(tk), vr = v_rsrc(tv);
    static_for<0, kMine>([&](auto p) { copy_k(kr, p, tk & 3); });
    static_for<0, kMine>([&](auto p) { copy_v(vr, p, tv & 3); });
  };
  constexpr int kStep = 2 * kMine;   // copies a step
  Lanes<HD> at;
  Soft<HD> soft;
  soft.clear();
  request(0, -2);
  request(1, -1);
  request(2, 0);
  request(3, 1);
  bf16x8 q[T::kT];
  load_row<HD>(a.q.p + (int64_t)(s.q0 + i) * a.q.t + head * a.q.h, i < s.nq, a.D, q);
  loaded();
  __builtin_amdgcn_s_barrier();
  fence();
  int t = 0;
  if (full >= 4) {
    uint32_t krow[T::kT], vtr[2][T::kD];
#pragma unroll
    for (int c = 0; c < T::kT; ++c) krow[c] = base + at.row(c);
#pragma unroll
    for (int d = 0; d < T::kD; ++d) {
      vtr[0][d] = base + kRing + at.tr(0, 0, d);
      vtr[1][d] = base + kRing + at.tr(1, 0, d);
    }
    auto k_op = [&](int slot, int c) { return *(const lds_bf16x8*)((lds_char*)(uintptr_t)krow[c] + slot * T::kBytes); };
    auto v_op = [&](int slot, int c) {   // product c: rows 16 (c / kD) .., channels 32 (c % kD) ..
      const int d = c % T::kD, off = slot * T::kBytes + 16 * (c / T::kD) * T::kRow;
      const i16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((lds_char*)(uintptr_t)vtr[0][d] + off));
      const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((lds_char*)(uintptr_t)vtr[1][d] + off));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    f32x16 sA, sB;
    bf16x8 pA[2], pB[2];
    sA = rows_times<HD>(lds, at, q);
    wait_and_sync_but<0>(true);   // every wave has read K(0): the first step's copies of K(4) go into its place
    {
      float mx = sA[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) mx = fmaxf(mx, sA[e]);
      soft.m = fmaxf(fmaf(pair_max(mx), a.c, kAbove), -3e38f);   // finite, also where infinities in K leave nothing of this tile
    }
    pB[0] = pB[1] = bf16x8{};
    const float c = a.c;
    // step T = t + SUB
    auto step = [&](auto sub_c, f32x16& s_cur, f32x16& s_nxt, bf16x8 (&p_prev)[2], bf16x8 (&p_cur)[2]) {
      constexpr int SUB = decltype(sub_c)::value, KS = (SUB + 1) & 3, VS = (SUB + 3) & 3;   // slots that are read
      constexpr int kRounds = 2 * T::kT, kExp = 16 / kRounds;
      const u32x4 kr = k_rsrc(t + SUB + 4), vr = v_rsrc(t + SUB + 2);
      bf16x8 kk[T::kT], vv[T::kT];
      const float negm = -soft.m;
      float x[16], sum[2];
      auto round = [&](auto i_c) {
        constexpr int I = decltype(i_c)::value;
        if constexpr (I == 0) {
          kk[0] = k_op(KS, 0);
          vv[0] = v_op(VS, 0);
          kk[1] = k_op(KS, 1);
          vv[1] = v_op(VS, 1);
        }
        static_for<2, T::kT>([&](auto j_c) {
          constexpr int J = decltype(j_c)::value;
          if constexpr ((2 * J - 4 > 0 ? 2 * J - 4 : 0) == I) {
            kk[J] = k_op(KS, J);
            vv[J] = v_op(VS, J);
          }
        });
        if constexpr (I < kRounds) {
          constexpr int C = I / 2;
          if constexpr (I % 2 == 0)
            s_nxt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kk[C], q[C], C > 0 ? s_nxt : f32x16{}, 0, 0, 0);
          else
            soft.acc[C % T::kD] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vv[C], p_prev[C / T::kD], soft.acc[C % T::kD], 0, 0, 0);
        }
        // the exponentials of the round before are summed and packed here, so that nothing waits for them
        if constexpr (I >= 1) {
#pragma unroll
          for (int e = 0; e < kExp; ++e) {
            constexpr int J0 = (I - 1) * kExp;
            const int J = J0 + e;
            if (J < 2) sum[J] = x[J];
            else sum[J & 1] += x[J];
            if (J & 1) {
              p_cur[J >> 3][(J & 7) - 1] = (bf16)x[J - 1];
              p_cur[J >> 3][J & 7] = (bf16)x[J];
              const u32x4 w = __builtin_bit_cast(u32x4, p_cur[J >> 3]);
              asm volatile("" ::"v"(w[(J & 7) >> 1]));   // packed here, and not sunk behind the branch below
            }
          }
        }
        if constexpr (I < kRounds) {
#pragma unroll
          for (int e = 0; e < kExp; ++e) x[I * kExp + e] = __builtin_amdgcn_exp2f(fmaf(s_cur[I * kExp + e], c, negm));
        }
        // a copy every few rounds
        constexpr int kEvery = kRounds / kStep;
        if constexpr (I % kEvery == 1 && I / kEvery < kStep) {
          constexpr int R = I / kEvery;
          if constexpr (R < kMine) copy_k(kr, std::integral_constant<int, R>{}, SUB);
          else copy_v(vr, std::integral_constant<int, R - kMine>{}, (SUB + 2) & 3);
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      static_for<0, kRounds + 1>(round);
      float part = sum[0] + sum[1];
      if (__ballot(!(part <= kRise)) != 0) {   // Soft::tile's rise, of the rows that need it
        acc_drain();
        float mx = s_cur[0];
#pragma unroll
        for (int e = 1; e < 16; ++e) mx = fmaxf(mx, s_cur[e]);
        const float to = pair_max(part) <= kRise ? soft.m : fmaxf(soft.m, fmaf(pair_max(mx), c, kAbove));
        const float by = __builtin_amdgcn_exp2f(soft.m - to);
        soft.m = to;
        soft.l *= by;
        part = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float y = __builtin_amdgcn_exp2f(fmaf(s_cur[e], c, -to));
          part += y;
          p_cur[e >> 3][e & 7] = (bf16)y;
        }
#pragma unroll
        for (int d = 0; d < T::kD; ++d)
#pragma unroll
          for (int e = 0; e < 16; ++e) soft.acc[d][e] *= by;
      }
      soft.l += part;
      __builtin_amdgcn_sched_barrier(0);
      wait_and_sync_but<2 * kStep>(false);   // K(T + 2) and V(T), requested two steps before, have landed
      __builtin_amdgcn_sched_barrier(0);
    };
    using C0 = std::integral_constant<int, 0>;
    using C1 = std::integral_constant<int, 1>;
    using C2 = std::integral_constant<int, 2>;
    using C3 = std::integral_constant<int, 3>;
    for (; t + 4 <= full; t += 4) {
      step(C0{}, sA, sB, pB, pA);
      step(C1{}, sB, sA, pA, pB);
      step(C2{}, sA, sB, pB, pA);
      step(C3{}, sB, sA, pA, pB);
    }
    add_packed<HD>(lds + kRing + 3 * T::kBytes, at, pB, soft.acc);   // V(t - 1)
    acc_drain();
  }
  // The tiles left: up to three whole ones, then those that some rows do not see all of. A step here reads K(t) and V(t), so K(t + 3)
  // is the furthest that it may request (the first one does so again).
  for (; t < tiles; ++t) {
    wait_and_sync_but<kStep>(false);
    request(t + 3, t + 2);
    lds_char* const kt = lds + (t & 3) * T::kBytes;
    if (t * kTile < lim_max) soft.template tile<true>(kt, kt + kRing, at, q, t * kTile, lim, lim_min, a.c);
  }
  if (i < s.nq) {
    const float l = pair_sum(soft.l);
    store_row<HD>(a.o.p + (int64_t)(s.q0 + i) * a.o.t + head * a.o.h, a.D, soft.acc, l == 0.f ? 0.f : 1.f / l);
    if (a.lse && g == 0)
      a.lse[(int64_t)head * a.tq + s.q0 + i] = lse_of(soft.m, l);
  }
  FVSR_WAIT_VM0();   // no copy outlives the workgroup's LDS
}

// ---- few queries a sequence: the keys split over the workgroups ------------------------------------------------------------
// A row is (query, head of the group), 32 to an item, so that K and V are read once for a group. All items' tiles of 32 keys
// stand in one order (sequence, key head, item, tile) and are cut into equal parts, one a workgroup, whatever the lengths are:
// a part begins and ends inside items, whose results it leaves for packed_join_kernel, and finishes those in between. Of an
// item's tiles each of the 4 waves takes every fourth, with a ring of its own and no barrier.
//
// Memory-bound: K and V move once. 24 sequences of up to 17280 keys, 16 heads of 128 over 4: 260 MB in 63 us, 4.1 TB/s, and 4.8 to join;
// one of 43200 keys, 12 heads over 2: 44 MB in 12.7 us and 4.3, where the offsets' two round trips, the rings' first tiles and the meeting
// of the waves in LDS stand beside the 9 that its bytes take. One workgroup a compute unit, with 128 KB of K and V under way or in use:
// three waves with rings of three tiles had the same bytes and took longer.
struct Parts {
  int work, parts;   // tiles of all items; workgroups that share them
  __device__ __forceinline__ int begin(int w) const { return (int)((int64_t)work * w / parts); }
  __device__ __forceinline__ int owner(int tile) const { return (int)((((int64_t)tile + 1) * parts - 1) / work); }
};
__device__ __forceinline__ int items_of(const PackedArgs& a, const Span& s) { return (s.nq * a.group + kTile - 1) / kTile; }
__device__ __forceinline__ int tiles_of(const Span& s) { return max(1, (s.nk + kTile - 1) / kTile); }
__device__ __forceinline__ Span lane_span(const PackedArgs& a, int b) {   // span_of, for a sequence of the lane's own
  return span_from(a, a.cu_q[b], a.cu_q[b + 1], a.cu_k[b], a.cu_k[b + 1], a.used_k ? a.used_k[b] : 0);
}

constexpr int kMaxParts = 256;        // workgroups of the split walk: its rings leave room for one on a compute unit
// Tiles a part, at the least (two a wave), but where items are shorter: each costs a round trip. One query over 4096 keys, 12 heads of
// 128: 11.4 us a call of a graph with 8, 13.2 with 4, 13.0 with 16; over 1024 keys and 2 key heads 11.3, 10.4 and 13.1.
constexpr int kMinTiles = 8;
constexpr int kMostWork = 1 << 30;    // tiles of a call (split)

// The parts, and for the tile `of(parts)` its sequence and that one's first tile. Called by the whole workgroup of 256;
// `sm` is LDS for 16 ints. The sequence is -1 where there is no such tile. Offsets that fall could make sequences overlap and
// their work pass 31 bits: none is done then.
template <class F>
__device__ __forceinline__ Parts find_tile(const PackedArgs& a, int* sm, F&& of, int& tile, int& b, int& first) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int per = (a.seqs + 255) / 256, b0 = min(tid * per, a.seqs), b1 = min(b0 + per, a.seqs);
  auto work_of = [&](int i) {
    const Span s = lane_span(a, i);
    return items_of(a, s) * tiles_of(s) * a.kv_heads;
  };
  int mine = 0;
  float about = 0.f, items = 0.f;
  for (int i = b0; i < b1; ++i) {
    const int n = work_of(i);
    mine += n;
    about += (float)n;
    items += (float)(items_of(a, lane_span(a, i)) * a.kv_heads);
  }
  about = wave_sum(about);
  items = wave_sum(items);
  int at = wave_scan_dpp(mine);
  if (lane == 63) {
    sm[wave] = at;
    sm[8 + wave] = __float_as_int(about);
    sm[12 + wave] = __float_as_int(items);
  }
  if (tid == 0) sm[4] = -1;
  __syncthreads();
  for (int w = 0; w < wave; ++w) at += sm[w];
  at -= mine;
  Parts p;
  p.work = uniform(sm[0] + sm[1] + sm[2] + sm[3]);
  about = __int_as_float(sm[8]) + __int_as_float(sm[9]) + __int_as_float(sm[10]) + __int_as_float(sm[11]);
  if (about > 1.5f * kMostWork) p.work = 0;
  items = __int_as_float(sm[12]) + __int_as_float(sm[13]) + __int_as_float(sm[14]) + __int_as_float(sm[15]);
  p.parts = max(1, min(a.max_parts, max(p.work / kMinTiles, uniform((int)fminf(items, 1e6f)))));
  tile = p.work > 0 ? of(p) : -1;
  if (tile >= at && tile < at + mine) {
    for (int i = b0; i < b1; ++i) {
      const int n = work_of(i);
      if (tile < at + n) {
        sm[4] = i;
        sm[5] = at;
        break;
      }
      at += n;
    }
  }
  __syncthreads();
  b = uniform(sm[4]);
  first = uniform(sm[5]);
  __syncthreads();
  return p;
}

// Partial results: of slot x, 32 rows of HD floats, then the rows' references and sums. In front of them, for each part, the item
// that begins in it and ends in a later one.
struct Cut {
  int pieces, inside;        // 0 pieces: no such item; whether the part begins before the item (its piece then is the second slot)
  int hk, r0, rows, q0;      // its key head, first row, rows in the sequence, and the sequence's first query
  int pad[2];
};
template <int HD>
struct Partial {
  static constexpr int kFloats = kTile * HD + 2 * kTile;
};

template <int HD>
__global__ __launch_bounds__(256, 1) void packed_split_kernel(PackedArgs a) {
  using T = Tile<HD>;
  __shared__ __attribute__((aligned(1024))) char smem[4][4 * T::kBytes];   // [wave][buffer][K, V]
  __shared__ float ml[4][2][kTile];
  __shared__ int sm[16];
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5, wave = uniform(tid >> 6);
  if (a.clear) {   // rows of no sequence, a head a turn
    const int lo = within(uniform(a.cu_q[0]), 0, a.tq), hi = within(uniform(a.cu_q[a.seqs]), lo, a.tq);
    for (int h = blockIdx.x; h < a.heads; h += gridDim.x) {
      if (a.clear & 1) {
        clear_rows(a.o, h, 0, lo, a.D);
        clear_rows(a.o, h, hi, a.tq, a.D);
      }
      if (a.lse)
        for (int r = tid; r < a.tq; r += 256)
          if (r < lo || r >= hi) a.lse[(int64_t)h * a.tq + r] = -INFINITY;
    }
  }
  int tile, b, first;
  const auto of = [&](const Parts& p) { return (int)blockIdx.x < p.parts ? p.begin(blockIdx.x) : -1; };
  const Parts parts = find_tile(a, sm, of, tile, b, first);
  Cut* const cut = (Cut*)a.part + blockIdx.x;
  float* const partial = a.part + kMaxParts * sizeof(Cut) / 4;
  if (tid == 0) cut->pieces = 0;
  if (b < 0) return;
  const int begin = tile, end = parts.begin(blockIdx.x + 1);
  const uint32_t base = lds_addr(smem[wave]);
  lds_char* const lds = (lds_char*)(uintptr_t)base;
  Lanes<HD> at;
  int koff[T::kCopies], voff[T::kCopies];
#pragma unroll
  for (int p = 0; p < T::kCopies; ++p) {
    koff[p] = copy_off<HD>(p, lane, (int)a.k.t * 2, a.D);
    voff[p] = copy_off<HD>(p, lane, (int)a.v.t * 2, a.D);
  }
  Span s = span_of(a, b);
  for (; tile < end;) {
    int items = items_of(a, s), tiles = tiles_of(s);
    while (tile - first >= items * tiles * a.kv_heads) {   // on to the next sequence; there is one, since tile < end <= work
      first += items * tiles * a.kv_heads;
      s = span_of(a, ++b);
      items = items_of(a, s);
      tiles = tiles_of(s);
    }
    const int unit = (tile - first) / tiles, t0 = (tile - first) - unit * tiles, t1 = min(tiles, t0 + end - tile);
    const int hk = unit / items, r0 = (unit - hk * items) * kTile, rows = s.nq * a.group;
    // the lane's row: query i, head h
    const int r = r0 + l32, i = min(r, rows - 1) / a.group, h = hk * a.group + min(r, rows - 1) % a.group;
    const int lim = keys_seen(a, s, i), full = keys_seen(a, s, r0 / a.group) / kTile;
    const bf16* const kb = a.k.p + (int64_t)s.k0 * a.k.t + hk * a.k.h;
    const bf16* const vb = a.v.p + (int64_t)s.k0 * a.v.t + hk * a.v.h;
    auto issue = [&](int t, int buf) {
      const u32x4 kr = rows_rsrc(kb, a.k.t, t * kTile, s.nk, a.D), vr = rows_rsrc(vb, a.v.t, t * kTile, s.nk, a.D);
      const uint32_t to = base + buf * 2 * T::kBytes;
      static_for<0, T::kCopies>([&](auto p) { dma16<p * 1024>(kr, to, koff[p], 0); });
      static_for<0, T::kCopies>([&](auto p) { dma16<p * 1024>(vr, to + T::kBytes, voff[p], 0); });
    };
    Soft<HD> soft;
    soft.clear();
    int buf = 0, t = t0 + wave;
    if (t < t1) issue(t, 0);
    bf16x8 q[T::kT];
    load_row<HD>(a.q.p + (int64_t)(s.q0 + i) * a.q.t + h * a.q.h, r < rows, a.D, q);
    loaded();
    auto step = [&](auto masked) {
      if (t + 4 < t1) {
        issue(t + 4, buf ^ 1);
        FVSR_WAIT_VM_LGKM0(2 * T::kCopies);
      } else {
        FVSR_WAIT_VM_LGKM0(0);
      }
      fence();
      lds_char* const kt = lds + buf * 2 * T::kBytes;
      soft.template tile<decltype(masked)::value>(kt, kt + T::kBytes, at, q, t * kTile, lim, 0, a.c);
      fence();
      FVSR_WAIT_VM_LGKM0(63);   // its reads are done before the next copies into this buffer
      t += 4;
      buf ^= 1;
    };
    while (t < min(full, t1)) step(std::false_type{});
    while (t < t1) step(std::true_type{});
    // the waves' results meet in LDS: each its rows x channels in its own ring
    {
      const float l = pair_sum(soft.l);
      if (g == 0) {
        ml[wave][0][l32] = soft.m;
        ml[wave][1][l32] = l;
      }
      float* const mine = (float*)smem[wave];
#pragma unroll
      for (int d = 0; d < T::kD; ++d)
#pragma unroll
        for (int c = 0; c < 4; ++c) {   // 16-byte pieces of a row, XOR-swizzled by row
          const int piece = (8 * d + 2 * c + g) ^ (l32 & 7);
          const auto& x = soft.acc[d];
          *(f32x4*)(mine + l32 * HD + 4 * piece) = f32x4{x[4 * c], x[4 * c + 1], x[4 * c + 2], x[4 * c + 3]};
        }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    float* const part = partial + (int64_t)(2 * blockIdx.x + (tile == begin ? 0 : 1)) * Partial<HD>::kFloats;
    if (tid == 0 && t0 == 0 && t1 < tiles)
      *cut = Cut{parts.owner(tile + tiles - 1) - (int)blockIdx.x + 1, tile > begin, hk, r0, rows, s.q0, {}};
    const int here = min(kTile, rows - r0);
    for (int e = tid; e < here * (HD / 4); e += 256) {
      const int row = e / (HD / 4), piece = e % (HD / 4);
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[w][0][row]);
      const float ref = m == -INFINITY ? 0.f : m;
      float l = 0.f;
      f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float by = __builtin_amdgcn_exp2f(ml[w][0][row] - ref), lw = ml[w][1][row];
        if (lw == 0.f) continue;   // a wave without keys for the row
        l = fmaf(lw, by, l);
        const f32x4 y = *(const f32x4*)((const float*)smem[w] + row * HD + 4 * (piece ^ (row & 7)));
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = fmaf(y[j], by, x[j]);
      }
      if (whole) {
        const int qi = (r0 + row) / a.group, qh = hk * a.group + (r0 + row) % a.group;
        const float by = l == 0.f ? 0.f : 1.f / l;
        if (4 * piece < a.D) {
          bf16x4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] = (bf16)(x[j] * by);
          *(bf16x4*)(a.o.p + (int64_t)(s.q0 + qi) * a.o.t + qh * a.o.h + 4 * piece) = o;
        }
        if (a.lse && piece == 0)
          a.lse[(int64_t)qh * a.tq + s.q0 + qi] = lse_of(m, l);
      } else {
        *(f32x4*)(part + row * HD + 4 * piece) = x;
        if (piece == 0) {
          part[kTile * HD + row] = m;
          part[kTile * HD + kTile + row] = l;
        }
      }
    }
    __syncthreads();
    tile += t1 - t0;
  }
}

// Workgroup (x, y): rows y, y + gridDim.y, .. of the item that begins in part x and ends in a later one. All of a row's pieces are
// asked for at once: their references and sums by a thread each, then their channels by 4 to a thread, the pieces dealt to the
// 256 / (HD / 4) groups of threads and joined in LDS. 4.3 us, a launch and three round trips; one row's pieces one after another took 60.
template <int HD>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedArgs a) {
  constexpr int kCols = HD / 4, kDeal = 256 / kCols;
  __shared__ float weight[kMaxParts];
  __shared__ float red[8];
  __shared__ __attribute__((aligned(16))) f32x4 sums[kDeal][kCols];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, x = blockIdx.x;
  const Cut cut = ((const Cut*)a.part)[x];
  if (cut.pieces <= 0) return;
  const int pieces = cut.pieces;   // <= kMaxParts
  const float* const partial = a.part + kMaxParts * sizeof(Cut) / 4;
  auto part = [&](int p) { return partial + (int64_t)(2 * (x + p) + (p == 0 ? cut.inside : 0)) * Partial<HD>::kFloats; };
  for (int row = blockIdx.y; row < min(kTile, cut.rows - cut.r0); row += gridDim.y) {
    __syncthreads();   // the row before is done with LDS
    float m = -INFINITY, l = 0.f;
    if (tid < pieces) {
      m = part(tid)[kTile * HD + row];
      l = part(tid)[kTile * HD + kTile + row];
    }
    float top = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if (lane == 0) red[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    // a piece without keys for the row counts for nothing
    const float by = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(m - (top == -INFINITY ? 0.f : top));
    if (tid < pieces) weight[tid] = by;
    l = wave_sum(l == 0.f ? 0.f : l * by);
    if (lane == 0) red[4 + wave] = l;
    __syncthreads();
    l = (red[4] + red[5]) + (red[6] + red[7]);
    const int col = tid % kCols, deal = tid / kCols;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int p = deal; p < pieces; p += kDeal) {
      const f32x4 y = *(const f32x4*)(part(p) + row * HD + 4 * col);
      const float w = weight[p];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = w == 0.f ? v[e] : fmaf(y[e], w, v[e]);
    }
    sums[deal][col] = v;
    __syncthreads();
    if (deal != 0) continue;
#pragma unroll
    for (int d = 1; d < kDeal; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += sums[d][col][e];
    const int qi = cut.q0 + (cut.r0 + row) / a.group, qh = cut.hk * a.group + (cut.r0 + row) % a.group;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (4 * col < a.D) {
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = (bf16)(v[e] * inv);
      *(bf16x4*)(a.o.p + (int64_t)qi * a.o.t + qh * a.o.h + 4 * col) = o;
    }
    if (a.lse && col == 0) a.lse[(int64_t)qh * a.tq + qi] = lse_of(top, l);
  }
}

// ---- backward ------------------------------------------------------------------------------------------------------------
// Two kernels, so that nothing is added with atomics: dQ walks over the keys like the forward pass (and leaves delta), dK and dV
// walk over the queries of the group's heads. Each makes S and dP again: 7 products in all where one kernel would make 5.
//
// dQ is bound like the forward pass: 2.20 ms, 1.25 PFLOP/s for its three products, the matrix core busy for 72 % of the cycles.
// What dK and dV need of a query beside its rows: -lse / scale and -delta, each as three bf16 numbers whose sum is the fp32 one.
// A product with ones adds them to S and dP in the matrix core: as operands of an addition they would have to be in 16 registers,
// read from LDS at eight times the bytes.
__device__ __forceinline__ bf16x8 stat_parts(float lse, float delta) {
  auto part = [](float& x) {
    const bf16 y = (bf16)x;
    x -= (float)y;
    return y;
  };
  const bf16 a = part(lse), b = part(lse), c = part(lse), d = part(delta), e = part(delta), f = part(delta);
  return bf16x8{a, b, c, (bf16)0.f, d, e, f, (bf16)0.f};
}

template <int HD>
__global__ __launch_bounds__(256, 2) void packed_dq_kernel(PackedArgs a) {
  using T = Tile<HD>;
  __shared__ __attribute__((aligned(1024))) char smem[8 * T::kBytes];   // [tile % 4][K, V]
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, wave = uniform(threadIdx.x >> 6);
  const int head = blockIdx.x % a.heads;
  Span s;
  const Block blk = block_of<false>(a, blockIdx.x / a.heads, s);
  if (a.clear) for_outside(blk, a.tq, [&](int lo, int hi) { clear_rows(a.dq, head, lo, hi, a.D); });
  if (blk.b < 0 || blk.b >= a.seqs) return;
  if (blk.row >= s.nq) return;
  const int i = blk.row + wave * 32 + l32, lim = keys_seen(a, s, i);
  const int lim_min = keys_seen(a, s, blk.row + wave * 32), lim_max = keys_seen(a, s, blk.row + wave * 32 + 31);
  // tiles that some row of the block sees, and that every one sees all of
  const int tiles = (keys_seen(a, s, blk.row + kRows - 1) + kTile - 1) / kTile, full = keys_seen(a, s, blk.row) / kTile;

  const bf16* const kb = a.k.p + (int64_t)s.k0 * a.k.t + head / a.group * a.k.h;
  const bf16* const vb = a.v.p + (int64_t)s.k0 * a.v.t + head / a.group * a.v.h;
  constexpr int kMine = T::kCopies / 4;
  int koff[kMine], voff[kMine];
#pragma unroll
  for (int p = 0; p < kMine; ++p) {
    koff[p] = copy_off<HD>(wave * kMine + p, lane, (int)a.k.t * 2, a.D);
    voff[p] = copy_off<HD>(wave * kMine + p, lane, (int)a.v.t * 2, a.D);
  }
  const uint32_t base = lds_addr(smem);
  lds_char* const lds = (lds_char*)(uintptr_t)base;
  auto issue = [&](int t) {
    const u32x4 kr = rows_rsrc(kb, a.k.t, t * kTile, s.nk, a.D), vr = rows_rsrc(vb, a.v.t, t * kTile, s.nk, a.D);
    const uint32_t to = base + (t & 3) * 2 * T::kBytes + wave * kMine * 1024;
    static_for<0, kMine>([&](auto p) {
      dma16<p * 1024>(kr, to, koff[p], 0);
      dma16<p * 1024>(vr, to + T::kBytes, voff[p], 0);
    });
  };
  if (tiles > 0) issue(0);
  if (tiles > 1) issue(1);
  bf16x8 q[T::kT], d_o[T::kT];
  load_row<HD>(a.q.p + (int64_t)(s.q0 + i) * a.q.t + head * a.q.h, i < s.nq, a.D, q);
  load_row<HD>(a.d_o.p + (int64_t)(s.q0 + i) * a.d_o.t + head * a.d_o.h, i < s.nq, a.D, d_o);
  float lse2 = 0.f, delta = 0.f;
  {
    bf16x8 o[T::kT];
    load_row<HD>(a.o.p + (int64_t)(s.q0 + i) * a.o.t + head * a.o.h, i < s.nq, a.D, o);
#pragma unroll
    for (int t = 0; t < T::kT; ++t)
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = fmaf((float)d_o[t][e], (float)o[t][e], delta);
    delta = pair_sum(delta);
    if (i < s.nq) lse2 = a.lse[(int64_t)head * a.tq + s.q0 + i] * kLog2e;
  }
  Lanes<HD> at;
  f32x16 acc[T::kD];
#pragma unroll
  for (int d = 0; d < T::kD; ++d) acc[d] = f32x16{};
  loaded();
  __builtin_amdgcn_s_barrier();   // tiles 0 and 1 have landed, for every wave
  fence();
  constexpr int kSlot = 2 * T::kBytes;
  const bool few = tiles <= 4;
  if (few) {
    // Where a row sees few keys, O is as large as V, and the rounding of O to bf16 would be a large part of what dS is off by: delta is
    // made of P and dP here, as the ring holds all the tiles. (Causal sequences of 17 to 4097 tokens: a gradient is at most 0.053 from a plain
    // form's, 0.093 without; the time is the same.) A sum of few dS is off by their rounding to bf16 as well; what that leaves is added
    // below. Over passes of 1 to 130 tokens the errors are 0.97 times what rounding the results costs (dK 1.00), where they were 1.37 times
    // and up to 1.55; 64 and 128 tokens of 12 heads take 19 and 30 us for 16 and 24.
    for (int t = 2; t < tiles; ++t) issue(t);
    wait_and_sync_but<0>(true);
    delta = 0.f;
    for (int t = 0; t < tiles; ++t) {
      const f32x16 x = rows_times<HD>(lds + t * kSlot, at, q), dp = rows_times<HD>(lds + t * kSlot + T::kBytes, at, d_o);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        delta += elem_row(e) < lim - t * kTile - 4 * g ? __builtin_amdgcn_exp2f(fmaf(x[e], a.c, -lse2)) * dp[e] : 0.f;
    }
    delta = pair_sum(delta);
  }
  if (i < s.nq && g == 0) {
    const int64_t to = (int64_t)head * a.tq + s.q0 + i;
    *(bf16x8*)(a.stat + 8 * to) = stat_parts(-a.lse[to] / a.scale, -delta);
  }
  uint32_t row[T::kT], tr[2][T::kD];
#pragma unroll
  for (int c = 0; c < T::kT; ++c) row[c] = base + at.row(c);
#pragma unroll
  for (int d = 0; d < T::kD; ++d) {
    tr[0][d] = base + at.tr(0, 0, d);
    tr[1][d] = base + at.tr(1, 0, d);
  }
  // operand x of a step on slot SLOT: rows of V (dP), rows of the next tile's K (its S), K transposed (dQ)
  auto operand = [&](auto slot, auto x) {
    constexpr int SLOT = decltype(slot)::value, X = decltype(x)::value, C = X % T::kT;
    if constexpr (X < T::kT) {
      return *(const lds_bf16x8*)((lds_char*)(uintptr_t)row[C] + SLOT * kSlot + T::kBytes);
    } else if constexpr (X < 2 * T::kT) {
      return *(const lds_bf16x8*)((lds_char*)(uintptr_t)row[C] + ((SLOT + 1) & 3) * kSlot);
    } else {
      constexpr int U = C / T::kD, D = C % T::kD, OFF = SLOT * kSlot + 16 * U * T::kRow;
      const i16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((lds_char*)(uintptr_t)tr[0][D] + OFF));
      const i16x4 z = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)((lds_char*)(uintptr_t)tr[1][D] + OFF));
      return __builtin_bit_cast(bf16x8, __builtin_shufflevector(y, z, 0, 1, 2, 3, 4, 5, 6, 7));
    }
  };
  f32x16 sA = f32x16{}, sB = f32x16{};
  if (tiles > 0) sA = rows_times<HD>(lds, at, q);
  int t = 0;
  // A step on a tile that every row sees whole: dP of it while its P is made, S of the next tile while dS is, then dQ; a product at a
  // time with a share of the rest behind it, as in packed_forward_kernel.
  auto step = [&](auto slot, f32x16& s_cur, f32x16& s_nxt) {
    constexpr int kRounds = 3 * T::kT, kAhead = 4, kExp = 16 / T::kT, kDs = (16 + T::kT - 3) / (T::kT - 2);
    const int tt = t + decltype(slot)::value + 3;
    const u32x4 kr = rows_rsrc(kb, a.k.t, tt * kTile, s.nk, a.D), vr = rows_rsrc(vb, a.v.t, tt * kTile, s.nk, a.D);
    constexpr uint32_t kTo = ((decltype(slot)::value + 3) & 3) * kSlot;
    bf16x8 op[kRounds], w[2];
    f32x16 dp;
    float p[16];
    auto round = [&](auto i_c) {
      constexpr int I = decltype(i_c)::value, C = I % T::kT;
      if constexpr (I == 0)
        static_for<0, kAhead>([&](auto x) { op[decltype(x)::value] = operand(slot, x); });
      if constexpr (I + kAhead < kRounds) op[I + kAhead] = operand(slot, std::integral_constant<int, I + kAhead>{});
      if constexpr (I < T::kT) {
        dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[I], d_o[C], C > 0 ? dp : f32x16{}, 0, 0, 0);
#pragma unroll
        for (int e = C * kExp; e < (C + 1) * kExp; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(s_cur[e], a.c, -lse2));
      } else if constexpr (I < 2 * T::kT) {
        s_nxt = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[I], q[C], C > 0 ? s_nxt : f32x16{}, 0, 0, 0);
        if constexpr (C >= 2) {   // the last product of dP takes two rounds
          constexpr int e0 = (C - 2) * kDs < 16 ? (C - 2) * kDs : 16, e1 = e0 + kDs < 16 ? e0 + kDs : 16;
#pragma unroll
          for (int e = e0; e < e1; ++e) w[e >> 3][e & 7] = (bf16)(p[e] * (dp[e] - delta));
        }
      } else {
        acc[C % T::kD] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(op[I], w[C / T::kD], acc[C % T::kD], 0, 0, 0);
        if constexpr (C % 2 == 0 && C / 2 < 2 * kMine) {
          constexpr int R = C / 2;
          if constexpr (R < kMine) dma16<R * 1024>(kr, base + kTo + wave * kMine * 1024, koff[R], 0);
          else dma16<(R - kMine) * 1024>(vr, base + kTo + T::kBytes + wave * kMine * 1024, voff[R - kMine], 0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    static_for<0, kRounds>(round);
    wait_and_sync_but<2 * kMine>(false);   // tile t + 2, requested a step before, has landed
    __builtin_amdgcn_sched_barrier(0);
  };
  if (tiles > 4) issue(2);
  if (!few && full >= 4) {
    wait_and_sync_but<2 * kMine>(false);
    for (; t + 4 <= full; t += 4) {
      step(std::integral_constant<int, 0>{}, sA, sB);
      step(std::integral_constant<int, 1>{}, sB, sA);
      step(std::integral_constant<int, 2>{}, sA, sB);
      step(std::integral_constant<int, 3>{}, sB, sA);
    }
    acc_drain();
  }
  // the tiles left: up to three whole ones, then those that some rows do not see all of
  auto last = [&](auto masked) {
    constexpr bool MASKED = decltype(masked)::value;
    wait_and_sync_but<2 * kMine>(t + 2 >= tiles);   // tiles t and t + 1 have landed (up to four all have)
    if (tiles > 4 && t + 3 < tiles) issue(t + 3);
    lds_char* const kt = lds + (t & 3) * kSlot;
    const int k0 = t * kTile;
    if (!MASKED || k0 < lim_max) {
      at.again();
      f32x16 dp = rows_times<HD>(kt + T::kBytes, at, d_o);
#pragma unroll
      for (int e = 0; e < 16; ++e) dp[e] = __builtin_amdgcn_exp2f(fmaf(sA[e], a.c, -lse2)) * (dp[e] - delta);
      if (MASKED) {
#pragma unroll
        for (int e = 0; e < 16; ++e) dp[e] = elem_row(e) < lim - k0 - 4 * g ? dp[e] : 0.f;
      }
      add_times<HD, MASKED>(kt, at, dp, 0, lim - k0, k0 + kTile <= lim_min, few, acc);
    }
    ++t;
    if (t < tiles) sA = rows_times<HD>(lds + (t & 3) * kSlot, at, q);
  };
  while (!few && t < full) last(std::false_type{});
  while (t < tiles) last(std::true_type{});
  FVSR_WAIT_VM0();   // no copy outlives the workgroup's LDS
  if (i < s.nq) store_row<HD>(a.dq.p + (int64_t)(s.q0 + i) * a.dq.t + head * a.dq.h, a.D, acc, a.scale);
}

// Two weights, from 0 to below 2, in 16 bits each: of fp32's bits the sign and the exponent's first are 0, the next 16 are kept, rounded.
// Off by at most 2^-10 of itself, a sixteenth of what rounding dS to bf16 costs in the mean square, down to 2^-126 (fp16 would lose the
// gradients of keys whose weights are all small; fp32 took twice the LDS, and the room for two tiles a step). NaN does not survive, but
// reaches dS by delta. Weights are below 2 because they are held to 2^0.5 where they are made: made again from a row's lse, one may pass 1 by
// what rounding does to large scores, by a factor of e and more from 2^24 on, and what passed 2 was lost from dK here. That minimum takes
// 1.0 to 1.5 % of the gradient; one of each weight as it is packed took 0.8 to 3, three-way maxima and a branch to it 0.8 to 1.5.
__device__ __forceinline__ uint32_t pack_weights(float lo, float hi) {
  return __builtin_amdgcn_perm((__float_as_uint(hi) << 2) + 0x8000u, (__float_as_uint(lo) << 2) + 0x8000u, 0x07060302u);
}
__device__ __forceinline__ float low_weight(uint32_t w) { return __uint_as_float((w & 0xffffu) << 14); }
__device__ __forceinline__ float high_weight(uint32_t w) { return __uint_as_float((w >> 16) << 14); }

// a part's sums of a block of keys, dK and dV; the parts of a block do not lie a power of two apart
template <int HD>
constexpr int kPartFloats = 2 * kRows * HD + 256;

// dK and dV of 128 keys: 8 waves, two to each 32 keys. One makes S, P and dV, the other, a tile of queries behind, dP, dS and dK
// from the P that the first one leaves in LDS (in 16 bits of its own, pack_weights).
// So a wave holds one operand and one sum, not two (which with S and dP beside them pass the 256 registers that two waves a SIMD
// have), and the two waves of a SIMD, one of each kind, are at the matrix core by turns.
//
// 3.25 ms, 1.13 PFLOP/s for its four products; the matrix core is busy for 57 % of the cycles, the rest are the barrier of a step and the
// reads behind it (3.18 without the minimum that holds weights below 2). Before that, steps of two tiles: 3.57 before the last round's blocks
// were cut (dkv_cut), 3.80 with steps of one. S and dP of the
// next tile before this one's rest, as the other kernels have it, was worth 2 % here and cost 40 % with 64 channels a head.
template <int HD>
__global__ __launch_bounds__(512, HD == 64 ? 4 : 2) void packed_dkv_kernel(PackedArgs a) {
  using T = Tile<HD>;
  // A step's tiles of queries: two, where they and their neighbours' fit (a step begins and ends with waiting), one where that leaves
  // room for a second workgroup on the compute unit.
  constexpr int kN = HD == 128 ? 2 : 1, kRowsN = kN * kTile, kSlots = kN == 2 ? 3 : 4, kEarly = kSlots - 2;
  constexpr int kSlot = 2 * kN * T::kBytes;                                               // Q, dO
  __shared__ __attribute__((aligned(1024))) char smem[kSlots * kSlot];                    // step n in slot n % kSlots
  __shared__ __attribute__((aligned(1024))) bf16x8 stat[kSlots][kN][64];                  // its rows' stat_parts
  __shared__ __attribute__((aligned(16))) u32x4 handed[2][4][kN][2][64];                  // P of step n in n % 2, a wave pair each
  const int lane = threadIdx.x & 63, l32 = lane & 31, g = lane >> 5, wave = uniform(threadIdx.x >> 6);
  const int pair = wave & 3;
  const bool makes_dv = wave < 4;
  // from block `dkv_whole` on, a block is cut
  const int over = max(0, (int)blockIdx.x - a.dkv_whole), parts = (int)blockIdx.x < a.dkv_whole ? 1 : a.dkv_parts;
  const int part = over % parts, block = (int)blockIdx.x - over + over / parts, hk = block % a.kv_heads;
  // the first keys, which most queries see, first
  Span s;
  const Block blk = block_of<true>(a, block / a.kv_heads, s);
  if (a.clear && part == 0)
    for_outside(blk, a.tk, [&](int lo, int hi) {
      clear_rows(a.dk, hk, lo, hi, a.D);
      clear_rows(a.dv, hk, lo, hi, a.D);
    });
  if (blk.b < 0 || blk.b >= a.seqs) return;
  if (blk.row >= s.room) return;
  const int j0 = blk.row + pair * 32, j = j0 + l32;
  const int off = s.nk - s.nq;   // causal: query i sees keys j <= i + off
  // The first query that sees a key of the block, down to a tile; the steps of a head from there on (none for keys that are not in
  // use), those before the first from which on every row sees all of the block, and those before the last one that may not be whole.
  const int q0 = a.causal ? min(s.nq, max(0, blk.row - off) / kTile * kTile) : 0;
  const int units = blk.row < s.nk ? (s.nq - q0 + kRowsN - 1) / kRowsN : 0;
  // where few queries see the block, what rounding P and dS to bf16 leaves is added as well: by the steps that may not be whole
  const bool few = s.nq - q0 <= kRows;
  const int u1 = few ? units : a.causal ? min(units, max(0, blk.row + kRows - 1 - off - q0 + kRowsN - 1) / kRowsN) : 0;
  const int u2 = max(u1, min(units, (s.nq - q0) / kRowsN));
  // of the steps of all the group's heads, those of this part: the first is `from_u` of head `from_h`
  const int all = units * a.group, begin = (int)((int64_t)all * part / parts);
  const int steps = (int)((int64_t)all * (part + 1) / parts) - begin;
  const int from_h = steps > 0 ? begin / units : 0, from_u = steps > 0 ? begin % units : 0;

  // a step's copies are dealt to the 8 waves: Q to the first 4, dO to the others
  constexpr int kMine = T::kCopies / 4;
  const HeadView<const bf16> from = makes_dv ? a.q : a.d_o;
  int voff[kMine];
#pragma unroll
  for (int p = 0; p < kMine; ++p) voff[p] = copy_off<HD>(pair * kMine + p, lane, (int)from.t * 2, a.D);
  const int soff = g == 0 ? l32 * 16 : (int)0x80000000;   // a tile's rows; the other lanes copy zeros
  const uint32_t base = lds_addr(smem) + (makes_dv ? 0 : kN * T::kBytes) + pair * kMine * 1024, sbase = lds_addr(stat);
  lds_char* const lds = (lds_char*)(uintptr_t)lds_addr(smem);
  Lanes<HD> at;
  f32x16 acc[T::kD];
#pragma unroll
  for (int d = 0; d < T::kD; ++d) acc[d] = f32x16{};
  // The step that is requested next: its rows, and those left of its head. Kept from one to the next, for a scalar multiplication or
  // two at the head of each step is a hundred cycles before the first product.
  int ih = hk * a.group + from_h, iu = from_u, in = 0, islot = 0;
  const bf16* rows = nullptr;
  const bf16* stats = nullptr;
  auto go_to = [&](int h, int u) {
    rows = from.p + (int64_t)(s.q0 + q0 + u * kRowsN) * from.t + h * from.h;
    stats = a.stat + ((int64_t)h * a.tq + s.q0 + q0 + u * kRowsN) * 8;
  };
  go_to(ih, iu);
  const int tile_bytes = kTile * (int)from.t * 2, rest = (s.nq - q0) % kRowsN;
  const int whole = ((kRowsN - 1) * (int)from.t + a.D) * 2, ragged = ((rest - 1) * (int)from.t + a.D) * 2;
  auto rsrc = [&](const bf16* at, int bytes) {
    return u32x4{(uint32_t)uniform((int)(uint32_t)(uint64_t)at), (uint32_t)uniform((int)((uint64_t)at >> 32 & 0xffffu)),
                 (uint32_t)uniform(bytes), 0x00020000u};
  };
  auto request = [&] {
    if (in < steps) {
      const bool end = iu == units - 1 && rest != 0;
      const u32x4 r = rsrc(rows, end ? ragged : whole);
#pragma unroll
      for (int k = 0; k < kN; ++k)
        static_for<0, kMine>([&](auto p) { dma16<p * 1024>(r, base + islot * kSlot + k * T::kBytes, voff[p], k * tile_bytes); });
      if (wave == 0) {
        const u32x4 sr = rsrc(stats, end ? rest * 16 : kRowsN * 16);
#pragma unroll
        for (int k = 0; k < kN; ++k) dma16<0>(sr, sbase + (islot * kN + k) * 1024, soff, k * kTile * 16);
      }
    }
    ++in;
    if (++islot == kSlots) islot = 0;
    rows += kRowsN * from.t;
    stats += kRowsN * 8;
    if (++iu == units) {
      iu = 0;
      go_to(++ih, iu);
    }
  };
  for (int n = 0; n < kEarly; ++n) request();
  const HeadView<const bf16> kv = makes_dv ? a.k : a.v;
  bf16x8 b[T::kT];
  load_row<HD>(kv.p + (int64_t)(s.k0 + j) * kv.t + hk * kv.h, j < s.nk, a.D, b);
  loaded();
  // the copies of kEarly - 1 steps may still be under way
  auto wait_for = [&](bool all) {
    fence();
    if (all || kEarly == 1) FVSR_WAIT_VM_LGKM0(0);
    else if (wave == 0) FVSR_WAIT_VM_LGKM0((kEarly - 1) * (kMine + 1) * kN);
    else FVSR_WAIT_VM_LGKM0((kEarly - 1) * kMine * kN);
    __builtin_amdgcn_s_barrier();
    fence();
  };
  // minus the rows' lse / scale (0) or delta (1), for every key: what S and dP of a tile begin with
  const bf16 one = (bf16)(g == 0 ? 1.f : 0.f), zero = (bf16)0.f;
  const bf16x8 ones = bf16x8{one, one, one, zero, zero, zero, zero, zero};
  auto minus = [&](int slot, int k, int which) {
    const bf16x4 x = *(const bf16x4*)((const char*)&stat[slot][k][l32] + 8 * which);
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_shufflevector(x, bf16x4{}, 0, 1, 2, 3, 4, 5, 6, 7), ones, f32x16{}, 0, 0, 0);
  };
  // the lane's key is seen by rows lo .. hi - 1 of a tile that begins with query r; whether any key of the wave is seen by the tile
  auto lo_of = [&](int r) { return a.causal ? j - off - r : 0; };
  auto hi_of = [&](int r) { return s.nq - r; };
  auto all_of = [&](int r) { return r + kTile <= s.nq && (!a.causal || j0 + 31 <= r + off); };
  auto any_of = [&](int r) { return r < s.nq && (!a.causal || j0 <= r + 31 + off); };
  auto first = [&](auto masked, int u, int n, int slot) {   // S, P and dV of step u of a head, the n-th of all
    constexpr bool MASKED = decltype(masked)::value;
    lds_char* const qt = lds + slot * kSlot;
    lds_char* const ot = qt + kN * T::kBytes;
    at.again();
    f32x16 p[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) p[k] = rows_times<HD>(qt + k * T::kBytes, at, b, minus(slot, k, 0));
    request();
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int r = q0 + u * kRowsN + k * kTile, lo = lo_of(r), hi = hi_of(r);
      if (MASKED && !any_of(r)) continue;   // neither here nor in `second`
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        p[k][e] = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(p[k][e] * a.c, 0.5f));   // NaN stays NaN
        if (MASKED) p[k][e] = elem_row(e) >= lo - 4 * g && elem_row(e) < hi - 4 * g ? p[k][e] : 0.f;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c)
        handed[n & 1][pair][k][c][lane] =
            u32x4{pack_weights(p[k][8 * c], p[k][8 * c + 1]), pack_weights(p[k][8 * c + 2], p[k][8 * c + 3]),
                  pack_weights(p[k][8 * c + 4], p[k][8 * c + 5]), pack_weights(p[k][8 * c + 6], p[k][8 * c + 7])};
      add_times<HD, MASKED>(ot + k * T::kBytes, at, p[k], lo, hi, all_of(r), few, acc);
    }
  };
  auto second = [&](auto masked, int u, int n, int slot) {   // dP, dS and dK of step u of a head, the n-th of all
    constexpr bool MASKED = decltype(masked)::value;
    lds_char* const qt = lds + slot * kSlot;
    lds_char* const ot = qt + kN * T::kBytes;
    at.again();
    f32x16 ds[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) ds[k] = rows_times<HD>(ot + k * T::kBytes, at, b, minus(slot, k, 1));
    request();
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int r = q0 + u * kRowsN + k * kTile, lo = lo_of(r), hi = hi_of(r);
      if (MASKED && !any_of(r)) continue;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const u32x4 p = handed[n & 1][pair][k][c][lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ds[k][8 * c + 2 * e] *= low_weight(p[e]);
          ds[k][8 * c + 2 * e + 1] *= high_weight(p[e]);
        }
      }
      if (MASKED) {
#pragma unroll
        for (int e = 0; e < 16; ++e) ds[k][e] = elem_row(e) >= lo - 4 * g && elem_row(e) < hi - 4 * g ? ds[k][e] : 0.f;
      }
      add_times<HD, MASKED>(qt + k * T::kBytes, at, ds[k], lo, hi, all_of(r), few, acc);
    }
  };
  // The walk of one kind of wave: `work` for each step of the part. The second kind is a step behind the first: `ahead` steps less are
  // left to be waited for.
  auto walk = [&](auto&& work, int ahead) {
    int u = from_u, slot = 0;
    for (int n = 0; n < steps;) {
      const int end = n + min(steps - n, units - u);   // to the head's last step
      auto run = [&](auto masked, int until) {
        for (; u < until && n < end; ++u, ++n) {
          wait_for(n + ahead >= steps);
          work(masked, u, n, slot);   // which requests a step
          if (++slot == kSlots) slot = 0;
        }
      };
      run(std::true_type{}, u1);
      run(std::false_type{}, u2);
      run(std::true_type{}, units);
      u = 0;
    }
  };
  if (makes_dv) {
    walk(first, 1);
    wait_for(true);
  } else {
    wait_for(1 >= steps);
    request();
    walk(second, 2);
  }
  if (j >= s.room) return;
  if (j >= s.nk) {   // not in use: seen by none
#pragma unroll
    for (int d = 0; d < T::kD; ++d) acc[d] = f32x16{};
  }
  if (parts > 1) {   // for packed_dkv_join_kernel: [block][part][dK, dV][key][HD]
    float* const sums = a.part + ((int64_t)(block - a.dkv_whole) * parts + part) * kPartFloats<HD>;
    float* const row = sums + ((makes_dv ? kRows : 0) + j - blk.row) * HD;
#pragma unroll
    for (int d = 0; d < T::kD; ++d)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        *(f32x4*)(row + 32 * d + 8 * c + 4 * g) = f32x4{acc[d][4 * c], acc[d][4 * c + 1], acc[d][4 * c + 2], acc[d][4 * c + 3]};
    return;
  }
  const HeadView<bf16> to = makes_dv ? a.dv : a.dk;
  store_row<HD>(to.p + (int64_t)(s.k0 + j) * to.t + hk * to.h, a.D, acc, makes_dv ? 1.f : a.scale);
}

// adds up the parts of dK and dV of a quarter of a block of keys, in their order
template <int HD>
__global__ __launch_bounds__(256) void packed_dkv_join_kernel(PackedArgs a) {
  const int block = a.dkv_whole + blockIdx.x, hk = block % a.kv_heads;
  Span s;
  const Block blk = block_of<true>(a, block / a.kv_heads, s);
  if (blk.b < 0 || blk.b >= a.seqs) return;
  constexpr int kCols = HD / 4, kEach = kRows / 4;
  const float* const parts = a.part + (int64_t)blockIdx.x * a.dkv_parts * kPartFloats<HD>;
#pragma unroll 2
  for (int e = threadIdx.x; e < 2 * kEach * kCols; e += 256) {
    const int col = e % kCols, row = (int)blockIdx.y * kEach + e / kCols % kEach, v = e / kCols / kEach, j = blk.row + row;
    if (j >= s.room || 4 * col >= a.D) continue;
    const float* p = parts + (v * kRows + row) * HD + 4 * col;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = 0; i < a.dkv_parts; ++i) {
      const f32x4 y = *(const f32x4*)(p + i * kPartFloats<HD>);
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] += y[c];
    }
    bf16x4 o;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = (bf16)(x[c] * (v ? 1.f : a.scale));
    const HeadView<bf16> to = v ? a.dv : a.dk;
    *(bf16x4*)(to.p + (int64_t)(s.k0 + j) * to.t + hk * to.h + 4 * col) = o;
  }
}

int64_t slots(int64_t rows, int seqs) { return rows / kRows + seqs + 1; }

// Whether the keys are split over the workgroups, or a workgroup walks over all keys of 128 queries of a head: by what each takes, in
// microseconds, for sequences of the average lengths. A walk of few blocks takes 0.39 us a tile of keys after 10; from 230 on they
// share the card. Split, there are two launches, and 256 workgroups take 0.24 us for each of the tiles of all items. That is from
// 12 heads of 128 over 12 and 2, 1 to 64 sequences of 1 to 1024 queries and 512 to 43200 keys: one query over 43200 keys 17 us
// split, 526 not; 256 queries 143 and 537; 1024 queries 489 and 547, over 4096 keys 83 and 66; 64 queries each of 64 sequences over
// 4096 keys, 12 heads over 2, 244 and 204, 32 queries 132 and 184. Heads of 64 channels go by the same figures, which were not taken for
// them. The lengths' products have to stay below kMostWork.
bool split(int seqs, int64_t tq, int64_t tk, int heads, int kv_heads) {
  const int64_t group = heads / kv_heads;
  if ((ceil_div(tq * group, kTile) + seqs) * (ceil_div(tk, kTile) + seqs) * kv_heads >= kMostWork) return false;
  const double tiles = (double)ceil_div(tk, (int64_t)kTile * seqs);
  const double items = (double)ceil_div(tq * group, (int64_t)kTile * seqs) * seqs * kv_heads;
  const double blocks = (double)ceil_div(tq, (int64_t)kRows * seqs) * seqs * heads;
  return 18 + items * tiles * (0.24 / kMaxParts) < 10 + 0.39 * tiles * std::max(1., blocks / 230);
}

}  // namespace

size_t packed_forward_workspace(int seqs, int64_t tq, int64_t tk, int heads, int kv_heads, int D) {
  if (!split(seqs, tq, tk, heads, kv_heads)) return 0;
  return kMaxParts * (sizeof(Cut) + 2 * sizeof(float) * (D <= 64 ? Partial<64>::kFloats : Partial<128>::kFloats));
}

int launch_packed_forward(PackedArgs a, void* ws, hipStream_t stream) {
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    if (split(a.seqs, a.tq, a.tk, a.heads, a.kv_heads)) {
      a.part = (float*)ws;
      a.max_parts = kMaxParts;
      const int64_t rows = std::min<int64_t>(kTile, ceil_div((int64_t)a.tq * a.group, a.seqs));   // a sequence's, on average
      hipLaunchKernelGGL((packed_split_kernel<HD>), dim3(kMaxParts), dim3(256), 0, stream, a);
      hipLaunchKernelGGL((packed_join_kernel<HD>), dim3(kMaxParts - 1, (unsigned)rows), dim3(256), 0, stream, a);
    } else {
      hipLaunchKernelGGL((packed_forward_kernel<HD>), dim3((unsigned)(slots(a.tq, a.seqs) * a.heads)), dim3(256), 0, stream, a);
    }
  };
  if (a.D <= 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

// Blocks of keys from `whole` on have their queries cut into `parts`, which costs a round trip of each part's sums through memory, so
// that a part is to have a few tens of steps: all blocks, where they are too few to fill the card, or those left over for a last round
// of workgroups, where all queries see all keys (causal, the last blocks are short), and the lengths of few sequences leave little doubt
// which blocks these are.
// Gradients cut and not cut, us: 16 heads of 64 over 4, causal sequences of 17 to 4097 tokens 279 and 425; 2048 tokens of 16 heads over 2,
// causal, 127 and 462; 17280 queries over 512 keys 261 and 513; 4096 tokens of 12 heads, causal, 267 and 234. With 512 blocks instead
// of kDkvBlocks 313, 124, 280, 252; with 2048 294, 126, 260, 304; with 16 or 64 steps within 10 %. Half of kDkvSteps where the blocks
// leave half of the card idle: 4, 490 and 895 tokens of 24 heads over 6, causal, 89 and 140; 669 of 32 over 8 59 and 79; 1024 of 12 63 and
// 63; a quarter 88, 68, 65; and of 192 blocks (2048 tokens of 12) half 122, all 100. The last round's blocks: 17280 tokens
// of 12 heads 5405 and 5647, of 64 channels 3109 and 3255; 4000, 5000 and 6000 tokens of 16 heads 1926 and 1951.
constexpr int kDkvBlocks = 1024, kDkvSteps = 32, kMostDkvParts = 16;
struct DkvCut {
  int64_t whole;
  int parts;
};
DkvCut dkv_cut(int seqs, int64_t tq, int64_t tk, int heads, int kv_heads, int D, bool causal) {
  if (tk == 0) return {0, 1};
  const int64_t blocks = (ceil_div(tk, kRows) + seqs / 2) * kv_heads;
  const int64_t steps = ceil_div(tq, (int64_t)kTile * seqs) * (heads / kv_heads);   // of a tile
  const int64_t most = std::min<int64_t>(steps / (blocks <= 128 ? kDkvSteps / 2 : kDkvSteps), kMostDkvParts);
  if (blocks < kDkvBlocks) return {0, (int)std::max<int64_t>(1, std::min(ceil_div(kDkvBlocks, blocks), most))};
  const int64_t at_once = D <= 64 ? 512 : 256, left = blocks % at_once;
  const int parts = causal || left == 0 || (int64_t)seqs * kv_heads >= at_once / 4 ? 1 : (int)std::min(at_once / left, most);
  return parts > 1 ? DkvCut{blocks - left, parts} : DkvCut{0, 1};
}
size_t stat_bytes(int64_t tq, int heads) { return ((size_t)tq * heads * 16 + 255) & ~(size_t)255; }

size_t packed_backward_workspace(int seqs, int64_t tq, int64_t tk, int heads, int kv_heads, int D, bool causal) {
  const DkvCut cut = dkv_cut(seqs, tq, tk, heads, kv_heads, D, causal);
  if (cut.parts == 1) return stat_bytes(tq, heads);
  const size_t parts = (size_t)(slots(tk, seqs) * kv_heads - cut.whole) * cut.parts;
  return stat_bytes(tq, heads) + parts * (D <= 64 ? kPartFloats<64> : kPartFloats<128>) * sizeof(float);
}

int launch_packed_backward(PackedArgs a, void* ws, hipStream_t stream) {
  a.stat = (bf16*)ws;
  a.part = (float*)((char*)ws + stat_bytes(a.tq, a.heads));
  const DkvCut cut = dkv_cut(a.seqs, a.tq, a.tk, a.heads, a.kv_heads, a.D, a.causal);
  a.dkv_parts = cut.parts;
  auto go = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    const unsigned blocks = (unsigned)(slots(a.tk, a.seqs) * a.kv_heads), whole = cut.parts > 1 ? (unsigned)cut.whole : blocks;
    a.dkv_whole = (int)whole;
    hipLaunchKernelGGL((packed_dq_kernel<HD>), dim3((unsigned)(slots(a.tq, a.seqs) * a.heads)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL((packed_dkv_kernel<HD>), dim3(whole + (blocks - whole) * cut.parts), dim3(512), 0, stream, a);
    if (whole < blocks) hipLaunchKernelGGL((packed_dkv_join_kernel<HD>), dim3(blocks - whole, 4), dim3(256), 0, stream, a);
  };
  if (a.D <= 64) go(std::integral_constant<int, 64>{});
  else go(std::integral_constant<int, 128>{});
  FVSR_HIP_CHECK(hipGetLastError());
  return FVSR_OK;
}

}  // namespace fvsr
