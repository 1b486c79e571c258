// Paged 16-bit KV cache: appending rows (with RoPE on the way) and exact causal attention over the pages, for several
// sequences of unlike lengths in one call.
//
// k, v [pages, Hkv, page, D] (page a power of two >= 16); table [B, W] names the page of rows [w page, (w + 1) page) of a
// sequence, an entry outside 0 .. pages - 1 names none (its rows are neither written nor attended); lens [B] counts a
// sequence's rows with the call's new ones, fresh [B] how many of the T token columns are real. Token j of a sequence is row
// lens - fresh + j and attends the rows up to its own.
#include "bb_common.h"
#include "bb_internal.h"

namespace bb {
namespace {

typedef __attribute__((address_space(3))) void lds_void;
typedef const __attribute__((address_space(4))) int32_t* const_i32;  // read by scalar loads
typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 bf16x4_t;
typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4_t;

template <bool V>
struct Constant {
  static constexpr bool value = V;
};

constexpr int kThreads = 256, kWaves = 4;
constexpr float kInf = __builtin_huge_valf();

template <bool F16>
BB_DEV float lo16(uint32_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu));
  else return __uint_as_float(w << 16);
}
template <bool F16>
BB_DEV float hi16(uint32_t w) {
  if constexpr (F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16));
  else return __uint_as_float(w & 0xffff0000u);
}

// ---------------------------------------------------------------------------------------------------------------
// The call's lengths. Everything a kernel indexes with goes through these: lens and fresh come from the caller's device
// memory and may hold anything.
BB_DEV int clampi(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
struct Sequence {
  int cap;    // rows that the table has entries for
  int n;      // rows, clamped to 0 .. cap
  int fresh;  // real token columns, 0 .. T
  int first;  // row of token 0 (may lie outside 0 .. cap - 1)
  // Rows that token j attends: the first seen(j) of them.
  BB_DEV int seen(int j) const { return j < fresh ? clampi(first + j + 1, 0, n) : 0; }
};
BB_DEV Sequence sequence(const PagedCache& c, int T, int b) {
  Sequence s;
  const int raw = c.lens[b];
  s.cap = c.W << c.page_log2;
  s.n = clampi(raw, 0, s.cap);
  s.fresh = c.fresh ? clampi(c.fresh[b], 0, T) : T;
  s.first = raw < -T ? -T : raw - s.fresh;
  return s;
}
// The page of row r (0 <= r < cap) of sequence b, or -1.
BB_DEV int page_of(const PagedCache& c, int b, int r) {
  const int e = c.table[b * c.st + (r >> c.page_log2)];
  return (uint32_t)e < (uint32_t)c.pages ? e : -1;
}

// ---------------------------------------------------------------------------------------------------------------
// RoPE of 8 elements x at dims d .. d + 7 and y at d + D / 2 .., in fp32, rounded once (HF's operator rounds each product
// and the sum to the element type).
struct Turn {
  float cx[8], sx[8], cy[8], sy[8];
};
template <bool F16>
BB_DEV void widen(const u32x4_t w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo16<F16>(w[i]);
    f[2 * i + 1] = hi16<F16>(w[i]);
  }
}
template <bool F16>
BB_DEV void load_turn(const PagedRope& r, int64_t at, int D, Turn& t) {
  if (r.f32) {
    const float* c = static_cast<const float*>(r.cos) + at;
    const float* s = static_cast<const float*>(r.sin) + at;
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const f32x4_t a = *reinterpret_cast<const f32x4_t*>(c + i), b = *reinterpret_cast<const f32x4_t*>(s + i);
      const f32x4_t e = *reinterpret_cast<const f32x4_t*>(c + D / 2 + i), f = *reinterpret_cast<const f32x4_t*>(s + D / 2 + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        t.cx[i + j] = a[j];
        t.sx[i + j] = b[j];
        t.cy[i + j] = e[j];
        t.sy[i + j] = f[j];
      }
    }
  } else {
    const uint16_t* c = static_cast<const uint16_t*>(r.cos) + at;
    const uint16_t* s = static_cast<const uint16_t*>(r.sin) + at;
    widen<F16>(ld16(c), t.cx);
    widen<F16>(ld16(s), t.sx);
    widen<F16>(ld16(c + D / 2), t.cy);
    widen<F16>(ld16(s + D / 2), t.sy);
  }
}
template <bool F16>
BB_DEV void rotate(const u32x4_t x, const u32x4_t y, const Turn& t, float (&p)[8], float (&q)[8]) {
  float a[8], b[8];
  widen<F16>(x, a);
  widen<F16>(y, b);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = fmaf(a[i], t.cx[i], -(b[i] * t.sx[i]));
    q[i] = fmaf(b[i], t.cy[i], a[i] * t.sy[i]);
    // (the asm keeps fp16 results single-rounded: the compiler would otherwise round the sum to fp16 by an fp16 fma)
    asm("" : "+v"(p[i]), "+v"(q[i]));
  }
}
template <bool F16>
BB_DEV void rotate(u32x4_t& x, u32x4_t& y, const Turn& t) {
  float p[8], q[8];
  rotate<F16>(x, y, t, p, q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = pack2<F16>(p[2 * i], p[2 * i + 1]);
    y[i] = pack2<F16>(q[2 * i], q[2 * i + 1]);
  }
}
// Two numbers as two 16-bit terms each.
template <bool F16>
BB_DEV u32x2_t two_terms(float a, float b) {
  uint32_t hi = pack2<F16>(a, b);
  asm("" : "+v"(hi));
  return u32x2_t{hi, pack2<F16>(a - lo16<F16>(hi), b - hi16<F16>(hi))};
}

// ---------------------------------------------------------------------------------------------------------------
// Append: K' = x cos + (-x[D/2:], x[:D/2]) sin of each new row into its page, V as it is, Q' beside. Bound by memory, each element
// read and written once. A lane takes 8 elements of a row's lower half and the 8 that RoPE pairs with them; a row is D / 16 lanes,
// rows go head by head (Q, then K, then V) through one token's, so that a wave's loads are contiguous in projections' outputs.
// 8111 tokens of 32 + 8 + 8 heads of 128, bf16: 204 MB in 33 us, 6.1 TB/s (a large copy: 5.1); one token of 64 sequences: 3.6 us.
template <int D, bool F16>
__global__ __launch_bounds__(kThreads) void paged_append_kernel(PagedAppendParams p) {
  constexpr int LPR = D / 16;
  const int heads = p.H + 2 * p.Hkv;
  const int64_t unit = (int64_t)blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int d = 8 * (threadIdx.x % LPR);
  if (unit >= (int64_t)p.B * p.T * heads) return;
  const int64_t token = unit / heads;
  const int head = (int)(unit - token * heads), b = (int)(token / p.T), j = (int)(token - (int64_t)b * p.T);
  const bool is_q = head < p.H, is_k = !is_q && head < p.H + p.Hkv;
  const uint16_t* src;
  uint16_t* dst;
  if (is_q) {
    src = p.q + b * p.sq0 + head * p.sq1 + j * p.sq2;
    dst = p.qout + b * p.so0 + head * p.so1 + j * p.so2;
  } else {
    const Sequence s = sequence(p.c, p.T, b);
    const int row = s.first + j;
    if (j >= s.fresh || row < 0 || row >= s.cap) return;
    const int page = page_of(p.c, b, row);
    if (page < 0) return;
    const int in = row & ((1 << p.c.page_log2) - 1);
    if (is_k) {
      const int g = head - p.H;
      src = p.k + b * p.sk0 + g * p.sk1 + j * p.sk2;
      dst = p.c.k + page * p.c.skp + g * p.c.skh + in * p.c.skr;
    } else {
      const int g = head - p.H - p.Hkv;
      src = p.v + b * p.sv0 + g * p.sv1 + j * p.sv2;
      dst = p.c.v + page * p.c.svp + g * p.c.svh + in * p.c.svr;
    }
  }
  u32x4_t x = ld16(src + d), y = ld16(src + d + D / 2);
  if ((is_q || is_k) && p.r.cos) {
    Turn t;
    load_turn<F16>(p.r, b * p.r.s0 + j * p.r.s1 + d, D, t);
    rotate<F16>(x, y, t);
  }
  st16(dst + d, x);
  st16(dst + d + D / 2, y);
}

// ---------------------------------------------------------------------------------------------------------------
// How a call's work is cut. A pair is (sequence, tile of VT query vectors of a KV head; vector v = token v / G, head v % G);
// its keys, the rows that its last real token attends, are cut into equal splits of whole units so that all splits of the
// call are about as long: `share` units, the call's total over p.target workgroups, at least p.min_share. Each workgroup
// finds its (pair, KV head, split) by the lengths on the device, and the grid goes by the capacity alone. Pairs with one split
// write the output, the others a partial for the merge.
BB_DEV int wave_scan(int v) {  // inclusive sum over the lanes
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
  return v;
}
BB_DEV int lane_int(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
// v / d for 0 <= v < 2^23, 0 < d, from a float reciprocal of d (a division of integers is some 40 instructions, and the code
// before the loops is run once, as its lines come in).
BB_DEV int quotient(int v, float inv, int d) {
  int q = (int)((float)v * inv);
  const int r = v - q * d;
  q = r < 0 ? q - 1 : r >= d ? q + 1 : q;
  return q;
}
BB_DEV int token_of(const PagedAttnParams& p, int v) { return quotient(v, p.inv_G, p.G); }
// Pair `pair` is tile pair_tile of sequence pair % B: the sequences' last tiles, which are the longest, come first.
BB_DEV int pair_tile(const PagedAttnParams& p, int pair) { return p.tiles == 1 ? 0 : p.tiles - 1 - quotient(pair, p.inv_B, p.B); }
BB_DEV int pair_sequence(const PagedAttnParams& p, int pair, int tile) { return pair - (p.tiles - 1 - tile) * p.B; }
// Rows that the pair's last real token attends (0: none of its tokens is real, or has rows).
BB_DEV int pair_keys(const PagedAttnParams& p, const Sequence& s, int tile) {
  const int j0 = token_of(p, tile * p.VT);
  int j1 = p.tiles == 1 ? p.T - 1 : token_of(p, tile * p.VT + p.VT - 1);
  if (j1 >= s.fresh) j1 = s.fresh - 1;
  return j1 < j0 ? 0 : s.seen(j1);
}
BB_DEV int pair_units(const PagedAttnParams& p, int pair) {
  if (pair >= p.pairs) return 0;
  const int tile = pair_tile(p, pair), k = pair_keys(p, sequence(p.c, p.T, pair_sequence(p, pair, tile)), tile);
  return (k + (1 << p.unit_log2) - 1) >> p.unit_log2;
}
// The share of a split, and the splits of a pair. Where the pairs fit a wave and the workgroups that run at once (p.fit_quarters >
// 0), the share is the F for which the call's splits are just no more than run at once, if F / least <= p.fit_quarters / 4 (5 / 4
// in tiles, where it so wastes little; any in the streaming kernel), and the rest of a pair is a split too; otherwise a pair's
// units over the least share are rounded, so that pairs a little over it stay whole. The share is never below the total over the
// workgroups aimed at, which the partials' space and the grid go by: a pair of several splits has at most twice its units over the
// share of them, so these are at most twice the workgroups aimed at, and all splits at most those and pairs * Hkv.
BB_DEV int sum_over_lanes(int v) { return lane_int(wave_scan(v), 63); }
struct Share {
  int units;
  bool fit;
  BB_DEV int splits(int u) const {
    const int n = quotient(fit ? u + units - 1 : u + units / 2, 1.0f / (float)units, units);
    return n > 0 || u == 0 ? n : 1;
  }
};
constexpr int kMostUnits = 1 << 22;  // of a pair, and so of a share: 2^28 rows of 64
BB_DEV Share share_of(const PagedAttnParams& p, int first, int64_t total) {
  const int64_t even = (total * p.Hkv + (1 << p.target_log2) - 1) >> p.target_log2;
  const int least = even < kMostUnits ? (int)even : kMostUnits;
  Share s{least > p.min_share ? least : p.min_share, false};
  if (p.fit_quarters > 0) {
    Share f{s.units, true};
    const int64_t bound = (int64_t)p.fit_quarters * s.units;  // looked at in between: each try is a scan, some 0.3 us
    while (4 * (int64_t)f.units <= bound && sum_over_lanes(f.splits(first)) * p.Hkv > 1 << p.target_log2)
      f.units += f.units < 8 ? 1 : f.units / 8;
    if (4 * (int64_t)f.units <= bound) s = f;
  }
  return s;
}
// What a workgroup does: split `split` of a pair, or (zero) the output of a pair without rows to attend, or nothing.
struct Item {
  bool live, zero;
  int b, tile, g, split, splits, slot;
};
// The item with index `item`, by a whole wave: the splits of all pairs in order, then the pairs without any, KV heads fastest.
// (Pairs without rows among the others would hold up the dispatch of long ones behind them.) Up to a wave's pairs it is found by a
// scan in each workgroup, 1.5 to 2 us at its start; more are laid out by a kernel before. (With scans of 64 at a time and with that
// kernel: 4 prompts of up to 2048 tokens, 128 pairs, 67 and 65 us; one token of 512 sequences of up to 512 rows 128 and 107, of
// 4096 of them 2429 and 824; 512 prompts of up to 128 tokens 732 and 349.)
BB_DEV Item find_item(const PagedAttnParams& p, int item, int lane) {
  Item it;
  if (p.items) {
    const int4 r = p.items[item];
    it.live = r.z > 0;
    it.zero = r.z == 0;
    it.b = __builtin_amdgcn_readfirstlane((uint32_t)r.x >> 16);
    it.g = __builtin_amdgcn_readfirstlane(r.x & 0xffff);
    it.tile = __builtin_amdgcn_readfirstlane(r.y);
    it.split = __builtin_amdgcn_readfirstlane(r.z & 0xffff);
    it.splits = __builtin_amdgcn_readfirstlane(r.z >> 16);
    it.slot = __builtin_amdgcn_readfirstlane(r.w);
  } else {
    const int u = pair_units(p, lane), total = sum_over_lanes(u);
    const int sp = share_of(p, u, total).splits(u), mine = sp * p.Hkv, split = sp > 1 ? mine : 0;
    const int upto = wave_scan(mine), slot_upto = wave_scan(split), items = lane_int(upto, 63);
    const uint64_t in = __builtin_amdgcn_ballot_w64(item < upto);
    it.live = in != 0;
    int pair = -1, splits = 0, slot = 0, before;
    if (it.live) {
      pair = __builtin_ctzll(in);
      splits = lane_int(sp, pair);
      slot = lane_int(slot_upto - split, pair);
      before = lane_int(upto - mine, pair);
    } else {
      const int nth = quotient(item - items, p.inv_Hkv, p.Hkv);
      before = items + nth * p.Hkv;
      const uint64_t none = __builtin_amdgcn_ballot_w64(lane < p.pairs && u == 0);
      const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(none >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)none, 0));
      if (nth < __builtin_popcountll(none)) pair = __builtin_ctzll(__builtin_amdgcn_ballot_w64((none >> lane & 1) && rank == nth));
    }
    it.zero = !it.live && pair >= 0;
    const int rest = item - before;
    it.split = it.live ? quotient(rest, p.inv_Hkv, p.Hkv) : 0;
    it.g = rest - it.split * p.Hkv;
    it.tile = pair_tile(p, pair < 0 ? 0 : pair);
    it.b = pair_sequence(p, pair < 0 ? 0 : pair, it.tile);
    it.splits = splits;
    it.slot = slot + it.g * splits + it.split;
    if (p.part && item == 0 && threadIdx.x == 0) p.plan[p.slots].x = lane_int(slot_upto, 63);
  }
  if (p.part && threadIdx.x == 0 && it.splits > 1)  // for the merge
    p.plan[it.slot] = make_int4(it.b, it.tile, it.g, it.split | it.splits << 16);
  return it;
}
// The same for more than a wave's pairs, in one workgroup: items[i] is (sequence << 16 | KV head, tile, split | splits << 16, slot),
// 0 splits for a pair without rows, -1 for nothing.
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PagedAttnParams p) {
  constexpr int WAVES = kPlanThreads / 64;
  __shared__ int sums[2][3][WAVES];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int turn = 0;
  // v[i]'s inclusive sums over the workgroup's threads up to this one, and over all of them.
  auto scan = [&](int (&v)[3], int (&all)[3]) {
    turn ^= 1;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      v[i] = wave_scan(v[i]);
      if (lane == 63) sums[turn][i][wave] = v[i];
    }
    __syncthreads();  // (the space of the scan before is not written again until all have read it: that is this barrier too)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      all[i] = 0;
      for (int w = 0; w < WAVES; ++w) {
        const int x = sums[turn][i][w];
        all[i] += x;
        v[i] += w < wave ? x : 0;
      }
    }
  };
  // A thread's units are a number of 34 bits (2^12 pairs of 2^22), summed in two parts.
  int64_t units = 0;
  for (int pair = tid; pair < p.pairs; pair += kPlanThreads) units += pair_units(p, pair);
  int v[3] = {(int)(units & 0xfffff), (int)(units >> 20), 0}, all[3];
  scan(v, all);
  const Share share = share_of(p, 0, ((int64_t)all[1] << 20) + all[0]);
  int items = 0, slots = 0, zeros = 0;
  for (int at = 0; at < p.pairs; at += kPlanThreads) {
    const int pair = at + tid, u = pair_units(p, pair), sp = share.splits(u), mine = sp * p.Hkv;
    v[0] = mine;
    v[1] = sp > 1 ? mine : 0;
    v[2] = 0;
    const int split = v[1];
    scan(v, all);
    if (sp > 0) {
      const int tile = pair_tile(p, pair), b = pair_sequence(p, pair, tile);
      const int first = items + v[0] - mine, slot = slots + v[1] - split;
      for (int s = 0; s < sp; ++s)
        for (int g = 0; g < p.Hkv; ++g) {
          const int i = first + s * p.Hkv + g;
          if (i < p.grid) p.items[i] = make_int4((int)((uint32_t)b << 16 | g), tile, s | sp << 16, slot + g * sp + s);
        }
    }
    items += all[0];
    slots += all[1];
  }
  for (int at = 0; at < p.pairs; at += kPlanThreads) {
    const int pair = at + tid;
    const bool none = pair < p.pairs && pair_units(p, pair) == 0;
    v[0] = none ? p.Hkv : 0;
    v[1] = v[2] = 0;
    scan(v, all);
    if (none) {
      const int tile = pair_tile(p, pair), b = pair_sequence(p, pair, tile), first = items + zeros + v[0] - p.Hkv;
      for (int g = 0; g < p.Hkv; ++g)
        if (first + g < p.grid) p.items[first + g] = make_int4((int)((uint32_t)b << 16 | g), tile, 0, 0);
    }
    zeros += all[0];
  }
  for (int i = items + zeros + tid; i < p.grid; i += kPlanThreads) p.items[i] = make_int4(0, 0, -1, 0);
  if (tid == 0 && p.part) p.plan[p.slots].x = slots;
}
// Zeros for a pair's tokens.
BB_DEV void store_zeros(const PagedAttnParams& p, const Item& it, int D, int tid, int threads) {
  for (int i = tid; i < p.VT * (D / 8); i += threads) {
    const int v = it.tile * p.VT + i / (D / 8), j = token_of(p, v), h = it.g * p.G + v - j * p.G;
    if (v < p.T * p.G) st16(p.out + it.b * p.so0 + h * p.so1 + j * p.so2 + 8 * (i % (D / 8)), u32x4_t{0, 0, 0, 0});
  }
}
// First unit of split s of u units in n splits: equal parts.
BB_DEV int split_begin(int u, int n, int s) { return n == 1 ? s * u : (int)((int64_t)u * s / n); }

// ---------------------------------------------------------------------------------------------------------------
// Attention of up to 16 NR query vectors of a KV head over a split of a sequence's rows: o = sum_i 2^(c q.k_i - m) v_i / sum_i
// 2^(c q.k_i - m), m the running maximum. Bound by memory, so the loads never wait for the arithmetic:
//   * Four waves, each with a stream of its own: chunks of 8 KB of K and 8 KB of V go straight into the wave's LDS by 16-byte
//     loads, non-temporal, through a buffer as long as the rows that there are (the rest lands as zeros). The next chunk's K goes
//     out when this one's is read, its V when this one's is, and exact vmcnt waits tell them apart. No barrier until the waves'
//     states meet. Two workgroups a CU have 128 KB in flight there.
//   * S^T = K Q^T leaves keys 16 kb + 4 a + i of vector x in lane (x, a), the order in which two transposed reads bring V's rows,
//     so the probabilities are operands of O^T = V^T P^T where they are.
//   * Splits go by the units of 4 chunks that there are, KV heads fastest, so that a head's pages stay with one XCD's L2.
// One token (4 query heads a KV head of 128, 8 KV heads, bf16) of 32 sequences of up to 8192 rows: 639 MB in 104 us and 2 of the
// merge behind it, 6.0 TB/s (a streaming read: 6.9); of one of 131072: 537 MB in 84 and 2. What is left is the start (launch,
// plan, table, first chunk: 9 us in which little is loaded) and XCDs that end up to 8 % apart.
template <bool F16>
BB_DEV f32x4_t mma16(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// A value over the four lanes x, x + 16, x + 32, x + 48 of a query vector.
BB_DEV float quarters_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return xhalf_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
BB_DEV float quarters_sum(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return xhalf_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}
BB_DEV void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// Eight bytes of LDS per lane: of 16 lanes, lanes 4 r .. 4 r + 3 point at 16 elements of row r, and lane l gets column l,
// row r in place r. (`restrict`: no load into LDS in flight writes what is read here; the compiler would wait for all of them.)
BB_DEV u32x2_t read_tr16(const uint8_t* __restrict__ at) {
  return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)at));
}

// A chunk's rows in LDS, 16 by 16, 2 D bytes each: 16-byte piece c of row r is at place c ^ k_swz(r) of its row, so that a
// fragment read (16 rows, one piece each of two neighbouring pieces) meets every bank once; V's swizzle keeps 32-byte
// blocks whole and spreads the eight rows that half a wave's transposed read touches.
template <int D>
BB_DEV int k_swz(int r) { return D == 128 ? r & 15 : (r >> 1) & 7; }
template <int D>
BB_DEV int v_swz(int r) { return D == 128 ? 2 * (r & 7) : 2 * ((r >> 1) & 3); }

// `rows` rows of a head's pages from row r on (all in one page) as a buffer of that size; empty for page < 0. (Everything here is
// one value a wave; the range by a minimum and selects alone: a clamp goes to the vector unit, and then each load is a loop over
// the values that its descriptor might have.)
struct PageRows {
  const char* at;
  uint32_t bytes;
};
BB_DEV PageRows page_rows(const PagedCache& c, bool is_v, const uint16_t* head, int page, int r, int rows, int row_bytes) {
  const uint32_t stride = (uint32_t)(is_v ? c.svr : c.skr) * 2, sp = (uint32_t)(is_v ? c.svp : c.skp);
  const uint32_t at = page < 0 ? 0u : (uint32_t)page;
  const uint32_t in = (uint32_t)(r & ((1 << c.page_log2) - 1)) * stride;
  uint32_t bytes = (uint32_t)(rows - 1) * stride + (uint32_t)row_bytes;
  bytes = page < 0 || rows <= 0 ? 0u : bytes;
  return PageRows{reinterpret_cast<const char*>(head) + (uint64_t)at * sp * 2 + in, bytes};
}

// 16 bytes a lane of those rows into LDS at `to` (one value a wave) + 16 lane.
template <int AUX>
BB_DEV void load_rows(const PageRows& at, uint8_t* to, uint32_t off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(
      __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(at.at), 0, (int)at.bytes, 0x00020000),
      reinterpret_cast<lds_void*>(reinterpret_cast<uintptr_t>(to)), 16, off, 0, 0, AUX);
}

// One wave's stream of chunks of KC rows, 8 KB of K and of V. AUX: of its loads, 2 (non-temporal) where a row is read once (32
// sequences of 8192 rows 107 us, 122 without), 0 where a head has several tiles and reads it again (a step of 64 vectors over 32768
// rows 54 us, 57 with; of 128 62 and 77).
template <int D, int AUX>
struct PageStream {
  static constexpr int KC = 4096 / D, GROUPS = KC / 16, LOADS = 8 / GROUPS;  // groups of 16 rows lie in one page
  static constexpr int RPL = 512 / D;                                        // rows of a load
  const PagedCache& c;
  const_i32 table;
  const uint16_t *kh, *vh;
  uint32_t row, kpiece, vpiece;
  int end;  // rows from here on are not read
  BB_DEV PageStream(const PagedCache& c_, int b, int g, int end_, int lane) : c(c_), end(end_) {
    table = (const_i32)(uintptr_t)(c.table + b * c.st);
    kh = c.k + g * c.skh;
    vh = c.v + g * c.svh;
    row = lane / (D / 8);
    kpiece = 16u * ((lane % (D / 8)) ^ k_swz<D>(row));
    vpiece = 16u * ((lane % (D / 8)) ^ v_swz<D>(row));
  }
  // The table's entries for the chunk at row k0 (not looked at yet: they are on their way) and the page of group j of it (-1:
  // none, or past the end).
  BB_DEV void entries(int k0, int (&e)[GROUPS]) const {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const int w = (k0 + 16 * j) >> c.page_log2;
      e[j] = table[w < c.W ? w : c.W - 1];
    }
  }
  BB_DEV void settle(int k0, int (&e)[GROUPS]) const {
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) e[j] = k0 + 16 * j < end && (uint32_t)e[j] < (uint32_t)c.pages ? e[j] : -1;
  }
  // Always eight loads, so that the counts the waits go by are exact; rows past the end and of no page land zeros.
  BB_DEV void fetch(bool is_v, uint8_t* to, int k0, const int (&e)[GROUPS]) const {
    const uint32_t rb = (uint32_t)(is_v ? c.svr : c.skr) * 2;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) {
      const int r = k0 + 16 * j;
      const PageRows at = page_rows(c, is_v, is_v ? vh : kh, e[j], r, end - r < 16 ? end - r : 16, 2 * D);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const uint32_t piece = is_v ? vpiece ^ 16u * v_swz<D>(RPL * i) : kpiece ^ 16u * k_swz<D>(RPL * i);
        load_rows<AUX>(at, to + 1024 * (LOADS * j + i), (row + RPL * i) * rb + piece);
      }
    }
  }
};

// A step's new rows among the rows [k0, k0 + KC) of a wave's landed chunk: rotated, into the pages and into LDS over what the
// pages held there. No other wave of the head's tile has these rows; where a head has several tiles, each does this for itself, and
// the pages get the same values from each.
template <int D, bool F16>
BB_DEV void patch_new_rows(const PagedAttnParams& p, const Sequence& s, int b, int g, int k0, int lane, uint8_t* ks, uint8_t* vs) {
  constexpr int KC = PageStream<D, 0>::KC, LPR = D / 16;
  const int d = 8 * (lane % LPR), c = lane % LPR;
  for (int i = lane / LPR; i < 2 * s.fresh; i += 64 / LPR) {
    const int j = i >> 1, row = s.first + j;
    const bool is_v = i & 1;
    if (row < k0 || row >= k0 + KC || row >= s.n) continue;
    const int page = page_of(p.c, b, row);
    if (page < 0) continue;
    const int64_t in = row & ((1 << p.c.page_log2) - 1);
    const uint16_t* src = is_v ? p.vnew + b * p.svn0 + g * p.svn1 + j * p.svn2 : p.knew + b * p.skn0 + g * p.skn1 + j * p.skn2;
    uint16_t* dst = is_v ? p.c.v + page * p.c.svp + g * p.c.svh + in * p.c.svr : p.c.k + page * p.c.skp + g * p.c.skh + in * p.c.skr;
    u32x4_t x = ld16(src + d), y = ld16(src + d + D / 2);
    if (!is_v && p.r.cos) {
      Turn t;
      load_turn<F16>(p.r, b * p.r.s0 + j * p.r.s1 + d, D, t);
      rotate<F16>(x, y, t);
    }
    st16(dst + d, x);
    st16(dst + d + D / 2, y);
    const int r = row - k0, z = is_v ? v_swz<D>(r & 15) : k_swz<D>(r & 15);
    uint8_t* to = (is_v ? vs : ks) + r * 2 * D;
    st16(to + 16 * (c ^ z), x);
    st16(to + 16 * ((c + LPR) ^ z), y);
  }
}

// A state's maximum is -inf where no row was attended, and kLowest where all scores were -inf or NaN: zeros are for the
// former only, the latter's sums of 0 or NaN make the quotient NaN, as its softmax is.
constexpr float kLowest = -3.4028234663852886e38f;
template <bool F16>
BB_DEV void store_output(const PagedAttnParams& p, int b, int g, int v, int d, f32x4_t O, float M, float L) {
  const int j = token_of(p, v), h = g * p.G + v - j * p.G;
#pragma unroll
  for (int k = 0; k < 4; ++k) O[k] = M == -kInf ? 0.0f : O[k] / L;
  *reinterpret_cast<u32x2_t*>(p.out + b * p.so0 + h * p.so1 + j * p.so2 + d) =
      u32x2_t{pack2<F16>(O[0], O[1]), pack2<F16>(O[2], O[3])};
}

// Values of V that are not finite, in a chunk that some vectors attend in part: a probability of 0 times an infinity would be
// NaN. They are taken out of the operand, and a vector that attends one is NaN in that column.
template <bool F16>
BB_DEV uint32_t not_finite(uint32_t w) {  // 0xffff in the halves that are not
  constexpr uint32_t e = F16 ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0xffffu : 0u) | ((w >> 16 & e) == e ? 0xffff0000u : 0u);
}
// What a column comes to whose values are not all finite goes by the values alone: +inf, -inf, or NaN where both or NaN are
// attended, however small their probabilities (which may be 0 as operands, and then make NaN of an infinity). So a sum that is not
// finite is looked up at its end: `pos` and `neg` are the first of the rows [begin, end) on a page whose value at d + k is +inf or
// NaN, -inf or NaN. (begin: a multiple of 4.)
constexpr int kNoRow = 0x7fffffff;
template <bool F16, int N>
BB_DEV void first_not_finite(const PagedCache& c, int b, const uint16_t* vh, int begin, int end, int d, int (&pos)[N], int (&neg)[N]) {
  constexpr uint32_t inf = F16 ? 0x7c00u : 0x7f80u;
#pragma unroll
  for (int k = 0; k < N; ++k) pos[k] = neg[k] = kNoRow;
#pragma unroll 1
  for (int r = begin; r < end; r += 4) {
    const int page = page_of(c, b, r);
    if (page < 0) continue;
    const uint16_t* v = vh + page * c.svp + (r & ((1 << c.page_log2) - 1)) * c.svr + d;
    uint16_t h[4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) h[i][k] = v[(r + i < end ? i : 0) * c.svr + k];
#pragma unroll
    for (int i = 3; i >= 0; --i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint32_t size = h[i][k] & 0x7fffu;
        const int row = size < inf ? kNoRow : r + i < end ? r + i : r;
        pos[k] = row < pos[k] && h[i][k] != (inf | 0x8000u) ? row : pos[k];
        neg[k] = row < neg[k] && h[i][k] != inf ? row : neg[k];
      }
  }
}
// `o` where the first `seen` rows are attended.
BB_DEV float with_infinities(float o, int pos, int neg, int seen) {
  if (pos < seen) o = neg < seen ? __builtin_nanf("") : kInf;
  else if (neg < seen) o = -kInf;
  return o;
}
template <int D, bool F16, int NR, bool NEW, int AUX>
__global__ __launch_bounds__(kThreads, 2) void paged_attn_kernel(PagedAttnParams p) {
  using Stream = PageStream<D, AUX>;
  constexpr int KC = Stream::KC, GROUPS = Stream::GROUPS, NDS = D / 32, NDB = D / 16;
  constexpr int ROW = D + 4;  // floats of a state's row: whole 16-byte pieces, rows on other banks
  __shared__ __attribute__((aligned(16))) uint8_t sm[kWaves][2][8192];
  const int tid = threadIdx.x, lane = tid & 63, x = lane & 15, a = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Item it = find_item(p, blockIdx.x, lane);
  if (it.zero) store_zeros(p, it, D, tid, kThreads);
  if (!it.live) return;
  const Sequence s = sequence(p.c, p.T, it.b);
  const int keys = __builtin_amdgcn_readfirstlane(pair_keys(p, s, it.tile));
  const int units = (keys + (1 << p.unit_log2) - 1) >> p.unit_log2;
  const int u0 = split_begin(units, it.splits, it.split), u1 = split_begin(units, it.splits, it.split + 1);
  int begin = u0 << p.unit_log2, end = u1 << p.unit_log2 < keys ? u1 << p.unit_log2 : keys;
  begin = __builtin_amdgcn_readfirstlane(begin);
  end = __builtin_amdgcn_readfirstlane(end);
  const int v0 = it.tile * p.VT;
  const int R = p.T * p.G - v0 < p.VT ? p.T * p.G - v0 : p.VT;

  const Stream in(p.c, it.b, it.g, end, lane);
  uint8_t *ks = sm[wave][0], *vs = sm[wave][1];
  int k0 = begin + wave * KC;
  int e[GROUPS], ne[GROUPS];
  in.entries(k0, e);
  // Q fragments: B operand of S^T = K Q^T, lane (x, a): dims 32 ds + 8 a .. of vector 16 r + x. Their loads go out before the
  // first chunk's, which they then need not wait for.
  u32x4_t qw[NR][NDS];
  int lim[NR], tok[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int v = 16 * r + x < R ? v0 + 16 * r + x : v0, j = token_of(p, v), h = it.g * p.G + v - j * p.G;
    tok[r] = j;
    lim[r] = 16 * r + x < R ? s.seen(j) : 0;
    const uint16_t* qr = p.q + it.b * p.sq0 + h * p.sq1 + j * p.sq2 + 8 * a;
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) qw[r][ds] = ld16(qr + 32 * ds);
  }
  __builtin_amdgcn_sched_barrier(0);
  in.settle(k0, e);
  in.fetch(false, ks, k0, e);
  in.fetch(true, vs, k0, e);
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) asm volatile("" : "+v"(qw[r][ds]));  // awaited here, not with the chunk before the loop
  // With new rows the rotated query is kept in two terms, as exact as fp32 products of it need; of 32 vectors in LDS, as two
  // workgroups a CU have no registers for it (one alone: 46 us where these take 39, 32 vectors over 32768 rows of 8 heads). All
  // waves write the same there, and each reads what it wrote or the same.
  constexpr int QT = NEW ? 2 : 1;
  constexpr bool AWAY = NEW && NR > 1;
  __shared__ __attribute__((aligned(16))) uint8_t qs[AWAY ? NR * NDS * QT * 1024 : 16];
  bf16x8_t qf[NR][AWAY ? 1 : NDS][QT];
  auto put_q = [&](int r, int ds, int i, u32x4_t w) {
    if constexpr (AWAY) st16(qs + 1024 * (QT * (NDS * r + ds) + i) + 16 * lane, w);
    else qf[r][ds][i] = as_bf16x8(w);
  };
  float scale[NR];  // of the scores
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    scale[r] = p.scale;
    if (NEW && p.r.cos) {
      float t[NDS][8];
#pragma unroll
      for (int ds = 0; ds < NDS / 2; ++ds) {
        Turn turn;
        load_turn<F16>(p.r, it.b * p.r.s0 + tok[r] * p.r.s1 + 32 * ds + 8 * a, D, turn);
        rotate<F16>(qw[r][ds], qw[r][ds + NDS / 2], turn, t[ds], t[ds + NDS / 2]);
      }
      if constexpr (F16) {  // a rotated query may lie past what fp16 holds: a power of two goes over to its scores' scale
        float top = 0.0f;
#pragma unroll
        for (int ds = 0; ds < NDS; ++ds)
#pragma unroll
          for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(t[ds][i]));
        if (__builtin_amdgcn_ballot_w64(top > 65504.0f)) {
          top = quarters_max(top);
          const int e = top > 65504.0f && top < kInf ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
          scale[r] = ldexpf(p.scale, e);
#pragma unroll
          for (int ds = 0; ds < NDS; ++ds)
#pragma unroll
            for (int i = 0; i < 8; ++i) t[ds][i] = ldexpf(t[ds][i], -e);
        }
      }
#pragma unroll
      for (int ds = 0; ds < NDS; ++ds) {
        u32x4_t w[2];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32x2_t two = two_terms<F16>(t[ds][2 * i], t[ds][2 * i + 1]);
          w[0][i] = two[0];
          w[1][i] = two[1];
        }
        put_q(r, ds, 0, w[0]);
        put_q(r, ds, 1, w[1]);
      }
    } else {
#pragma unroll
      for (int ds = 0; ds < NDS; ++ds) {
        put_q(r, ds, 0, qw[r][ds]);
        if constexpr (NEW) put_q(r, ds, 1, u32x4_t{0, 0, 0, 0});
      }
    }
  }
  // the fewest rows that a token of the tile attends: chunks below need no mask (what padding gets there is not stored)
  const int fewest = __builtin_amdgcn_readfirstlane(s.seen(token_of(p, v0)));

  float m[NR], l[NR];
  bool seen[NR];
  f32x4_t o[NR][NDB];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    m[r] = -kInf;
    l[r] = 0.0f;
    seen[r] = false;
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[r][db] = f32x4_t{0, 0, 0, 0};
  }
  uint32_t kread[NDS], vread[2];  // fragment reads: key block kb is 32 D kb bytes on (both swizzles repeat every 16 rows)
#pragma unroll
  for (int ds = 0; ds < NDS; ++ds) kread[ds] = 2 * D * x + 16 * ((4 * ds + a) ^ k_swz<D>(x));
  const int vrow = 4 * a + (x >> 2);  // of 16: the lane's row and 8-byte piece x & 3 of a 32-byte block

  for (; k0 < end; k0 += kWaves * KC) {
    in.entries(k0 + kWaves * KC, ne);
    __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): this chunk's K has landed, its V may be in flight
    wave_fence();
    if (NEW && k0 + KC > s.first && k0 < s.n) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // V too
      wave_fence();
      patch_new_rows<D, F16>(p, s, it.b, it.g, k0, lane, ks, vs);
      __builtin_amdgcn_s_waitcnt(0x0070);  // all done: the counts below hold
      wave_fence();
    }
    f32x4_t y[NR][KC / 16];
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int kb = 0; kb < KC / 16; ++kb) y[r][kb] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int ds = 0; ds < NDS; ++ds) {
      if constexpr (AWAY)
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int t = 0; t < QT; ++t)
            qf[r][0][t] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(qs + 1024 * (QT * (NDS * r + ds) + t) + 16 * lane));
#pragma unroll
      for (int kb = 0; kb < KC / 16; ++kb) {
        const bf16x8_t kf = as_bf16x8(*reinterpret_cast<const u32x4_t*>(ks + kread[ds] + 32 * D * kb));
#pragma unroll
        for (int r = 0; r < NR; ++r)
#pragma unroll
          for (int t = 0; t < QT; ++t) y[r][kb] = mma16<F16>(kf, qf[r][AWAY ? 0 : ds][t], y[r][kb]);
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): K is read, its space is free
    wave_fence();
    __builtin_amdgcn_sched_barrier(0);  // (the table's entries are wanted from here on, not before the products)
    in.settle(k0 + kWaves * KC, ne);
    in.fetch(false, ks, k0 + kWaves * KC, ne);

    bool whole = k0 + KC <= fewest;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) whole = whole && e[j] >= 0;
    bf16x8_t pf[NR][KC / 32][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
#pragma unroll
      for (int kb = 0; kb < KC / 16; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) y[r][kb][i] *= F16 && NEW ? scale[r] : p.scale;
      if (whole) {
        seen[r] = true;
      } else {
#pragma unroll
        for (int kb = 0; kb < KC / 16; ++kb) {
          const int stop = e[kb] < 0 ? 0 : lim[r], row = k0 + 16 * kb;
          seen[r] |= row < stop;
#pragma unroll
          for (int i = 0; i < 4; ++i) y[r][kb][i] = row + 4 * a + i < stop ? y[r][kb][i] : -kInf;
        }
      }
      float mx = y[r][0][0];
#pragma unroll
      for (int kb = 0; kb < KC / 16; ++kb)
#pragma unroll
        for (int i = 0; i < 4; ++i) mx = fmaxf(mx, y[r][kb][i]);
      const float mn = fmaxf(m[r], quarters_max(mx));
      if (__builtin_amdgcn_ballot_w64(mn > m[r])) {
        const float alpha = mn > m[r] ? fast_exp2(m[r] - mn) : 1.0f;
        m[r] = mn;
        l[r] *= alpha;
#pragma unroll
        for (int db = 0; db < NDB; ++db)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[r][db][i] *= alpha;
      }
      const float off = m[r] == -kInf ? 0.0f : m[r];
#pragma unroll
      for (int st = 0; st < KC / 32; ++st) {
        float pr[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pr[i] = fast_exp2(y[r][2 * st + i / 4][i % 4] - off);
          l[r] += pr[i];
        }
        // in two terms: with one, the probabilities' rounding would be as large as the output's own, which is all the error that
        // there is otherwise (and the matrix cores idle here)
        u32x4_t hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const u32x2_t t = two_terms<F16>(pr[2 * i], pr[2 * i + 1]);
          hi[i] = t[0];
          lo[i] = t[1];
        }
        pf[r][st][0] = as_bf16x8(hi);
        pf[r][st][1] = as_bf16x8(lo);
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0F78);  // vmcnt(8): this chunk's V has landed, the next K may be in flight
    wave_fence();
    const auto values = [&](auto part) {
#pragma unroll
      for (int st = 0; st < KC / 32; ++st)
#pragma unroll
        for (int db = 0; db < NDB; ++db) {
          const uint32_t at = 2 * D * vrow + 16 * ((2 * db + ((x >> 1) & 1)) ^ v_swz<D>(vrow)) + 8 * (x & 1);
          const u32x2_t w0 = read_tr16(vs + 64 * D * st + at), w1 = read_tr16(vs + 64 * D * st + 32 * D + at);
          u32x4_t vw = {w0[0], w0[1], w1[0], w1[1]};
          if constexpr (decltype(part)::value) {
            u32x4_t bad;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              bad[i] = not_finite<F16>(vw[i]);
              vw[i] &= ~bad[i];
            }
            if (__builtin_amdgcn_ballot_w64((bad[0] | bad[1] | bad[2] | bad[3]) != 0)) {
              constexpr uint32_t one = F16 ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
              for (int r = 0; r < NR; ++r) {
                u32x4_t att;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int kb = 2 * st + i / 2, key = k0 + 16 * kb + 4 * a + 2 * (i % 2);
                  att[i] = e[kb] < 0 ? 0u : (key < lim[r] ? one & 0xffffu : 0u) | (key + 1 < lim[r] ? one & 0xffff0000u : 0u);
                }
                const f32x4_t hits = mma16<F16>(as_bf16x8(u32x4_t{bad[0] & one, bad[1] & one, bad[2] & one, bad[3] & one}),
                                                as_bf16x8(att), f32x4_t{0, 0, 0, 0});
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (hits[i] > 0.0f) o[r][db][i] = __builtin_nanf("");
              }
            }
          }
          const bf16x8_t vf = as_bf16x8(vw);
#pragma unroll
          for (int r = 0; r < NR; ++r)
#pragma unroll
            for (int t = 0; t < 2; ++t) o[r][db] = mma16<F16>(vf, pf[r][st][t], o[r][db]);
        }
    };
    // (one token attends all rows that were read)
    if (whole || p.T == 1) values(Constant<false>{});
    else values(Constant<true>{});
    __builtin_amdgcn_s_waitcnt(0xC07F);
    wave_fence();
    in.fetch(true, vs, k0 + kWaves * KC, ne);
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) e[j] = ne[j];
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // nothing lands in LDS any more

  // The four waves' states under one maximum.
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    __syncthreads();
    float* f = reinterpret_cast<float*>(&sm[0][0][0]) + (wave * 16 + x) * ROW;
    const float ls = quarters_sum(l[r]);
#pragma unroll
    for (int db = 0; db < NDB; ++db) *reinterpret_cast<f32x4_t*>(f + 16 * db + 4 * a) = o[r][db];
    if (a == 0) {
      f[D] = !seen[r] || lim[r] <= 0 ? -kInf : m[r] == -kInf ? kLowest : m[r];
      f[D + 1] = ls;
    }
    __syncthreads();
    for (int i = tid; i < 16 * (D / 4); i += kThreads) {
      const int vv = 16 * r + i / (D / 4), d = 4 * (i % (D / 4));
      if (vv >= R) continue;
      const float* g = reinterpret_cast<const float*>(&sm[0][0][0]) + (i / (D / 4)) * ROW;
      float M = -kInf, L = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, g[w * 16 * ROW + D]);
      const float off = M == -kInf ? 0.0f : M;
      f32x4_t O = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float* f = g + w * 16 * ROW;
        const float wt = fast_exp2(f[D] - off);
        const f32x4_t t = *reinterpret_cast<const f32x4_t*>(f + d);
        L = fmaf(wt, f[D + 1], L);
#pragma unroll
        for (int k = 0; k < 4; ++k) O[k] = fmaf(wt, t[k], O[k]);
      }
      if (!(fabsf(O[0]) + fabsf(O[1]) + fabsf(O[2]) + fabsf(O[3]) < kInf) && L > 0.0f && L < kInf) {
        int pos[4], neg[4];
        first_not_finite<F16>(p.c, it.b, p.c.v + it.g * p.c.svh, begin, end, d, pos, neg);
        const int attended = s.seen(token_of(p, v0 + vv));
#pragma unroll
        for (int k = 0; k < 4; ++k) O[k] = with_infinities(O[k], pos[k], neg[k], attended);
      }
      if (it.splits == 1) {
        store_output<F16>(p, it.b, it.g, v0 + vv, d, O, M, L);
      } else {
        float* dst = p.part + ((int64_t)it.slot * p.VT + vv) * ROW;
        *reinterpret_cast<f32x4_t*>(dst + d) = O;
        if (d == 0) {
          dst[D] = M;
          dst[D + 1] = L;
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Attention of many query vectors (prompts and their chunks): bound by the matrix cores and what feeds them, so a workgroup's 8
// waves share every K and V tile of 64 rows, 32 vectors each (two blocks of 16, so that every fragment read from LDS feeds two
// products).
//   * Waves w and w + 4 share a SIMD and run half a tile apart: while one does products (O^T += V^T P^T of the tile before,
//     then S^T = K Q^T), the other does its softmax, with workgroup barriers in between.
//   * Tiles stream through rings of four stages by 16-byte loads into LDS, two tiles before they are wanted; each load's rows lie in
//     one page, whose table entry came by a scalar load a tile earlier.
//   * S^T leaves keys 16 kb + 4 a + i of vector x in lane (x, a), which is the order in which two transposed reads bring V's
//     rows, so the probabilities are operands where they are.
//   * The exponent's offset moves only when a probability would pass 2^8. Tiles that some vector attends in part, and every tile
//     of a split whose table names no page somewhere, take a mask; they come last.
// 4096 tokens of 32 heads of 128 (8 KV heads) over 32768 rows, bf16: 1605 us, 1285 TFLOP/s (a large product: 1256), 1.7 us a tile
// and workgroup at a clock that the power holds at 1.9 to 2.0 GHz; the matrix cores are busy 60 % of it, the LDS reads of 256 KB a
// tile (8 waves x 32 KB) take about as long as the products. head_dim 64, fp16: 1080 us, 954 TFLOP/s, 1.26 us a tile: as many
// exponentials for half the products. Shapes tried there: four waves of 32 vectors, three workgroups a CU and one barrier a tile,
// 1150 us (four prompts of 2048 tokens 63 against 64); eight waves with one barrier a tile 1210; the row sums by products with ones
// 1090; two workgroups of eight waves a CU (128 registers) spill.
constexpr int kTileWaves = 8, kTileStages = 4, kTileVecs = 32 * kTileWaves, kTileRows = 64;
constexpr float kOver = 256.0f;  // 2^8

template <int D>
struct TileLds {
  static constexpr int BYTES = kTileRows * D * 2;         // of a K or V tile
  static constexpr int LOADS = BYTES / 1024 / kTileWaves;  // of a wave: 2 or 1
  static constexpr int RPL = 512 / D;                      // rows of a load
};

// The loads of a wave's part of a tile. ONE: pages of 64 rows and more, so a tile lies in one page and a descriptor serves all of a
// wave's loads of it (with smaller pages each load has its own: some 130 scalar instructions a tile instead of 40, in the phase
// that the matrix cores wait for).
template <int D, bool ONE>
struct TileLoader {
  using L = TileLds<D>;
  static constexpr int PAGES = ONE ? 1 : L::LOADS;
  const PagedCache& c;
  const_i32 table;
  const uint16_t *kh, *vh;
  uint32_t koff[L::LOADS], voff[L::LOADS];
  int row0, end;  // first row of the wave's first load in a tile; rows from `end` on are not read
  BB_DEV TileLoader(const PagedCache& c_, int b, int g, int end_, int wave, int lane) : c(c_), end(end_) {
    table = (const_i32)(uintptr_t)(c.table + b * c.st);
    kh = c.k + g * c.skh;
    vh = c.v + g * c.svh;
    row0 = L::RPL * wave;
    const int row = lane / (D / 8), piece = lane % (D / 8);
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
      const int r = row0 + row + L::RPL * kTileWaves * i, at = ONE ? r : row;
      koff[i] = at * (uint32_t)c.skr * 2 + 16 * (piece ^ k_swz<D>(r & 15));
      voff[i] = at * (uint32_t)c.svr * 2 + 16 * (piece ^ v_swz<D>(r & 15));
    }
  }
  BB_DEV int entry(int r) const {  // of row r's page
    const int w = r >> c.page_log2;
    return table[w < c.W ? w : c.W - 1];
  }
  struct Entries {
    int e[PAGES];
  };
  BB_DEV Entries entries(int k0) const {
    Entries x;
#pragma unroll
    for (int i = 0; i < PAGES; ++i) x.e[i] = entry(k0 + (ONE ? 0 : row0 + L::RPL * kTileWaves * i));
    return x;
  }
  // This wave's part of the K or V tile of rows k0 .., into `to`: always LOADS loads; rows past the end and of no page land zeros.
  BB_DEV void load(bool is_v, uint8_t* to, int wave, int k0, const Entries& x) const {
    constexpr int ROWS = ONE ? kTileRows : L::RPL;
    PageRows at;
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
      if (i < PAGES) {
        const int r = ONE ? k0 : k0 + row0 + L::RPL * kTileWaves * i;
        const int page = (uint32_t)x.e[i] < (uint32_t)c.pages ? x.e[i] : -1;
        at = page_rows(c, is_v, is_v ? vh : kh, page, r, end - r < ROWS ? end - r : ROWS, 2 * D);
      }
      load_rows<0>(at, to + 1024 * (wave + kTileWaves * i), is_v ? voff[i] : koff[i]);
    }
  }
};

// Workgroup barrier that does not drain the loads in flight (the ring publishes them by explicit vmcnt waits); nothing moves
// across it.
BB_DEV void ring_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
// The waves of a workgroup see what this one stored in LDS behind the next ring_barrier, which waits for no store by itself.
// (A release fence waits for the loads in flight too.)
BB_DEV void publish() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
BB_DEV uint32_t lds_addr(const void* p) {
  return (uint32_t)reinterpret_cast<uintptr_t>(
      reinterpret_cast<__attribute__((address_space(3))) const void*>(reinterpret_cast<uintptr_t>(p)));
}
BB_DEV u32x4_t lds16(uint32_t at) { return *(const __attribute__((address_space(3))) u32x4_t*)(uintptr_t)at; }
BB_DEV u32x2_t lds_tr16(uint32_t at) {
  return read_tr16((const uint8_t*)(const __attribute__((address_space(3))) uint8_t*)(uintptr_t)at);
}

template <int D>
struct TileState {
  bf16x8_t qf[2][D / 32];  // Q^T: vector block rb, 32 dims
  f32x4_t o[D / 16][2];    // O^T: dims 16 db + 4 a + i of vector 16 rb + x
  f32x4_t s[4][2];         // S^T of the current tile: keys 16 kb + 4 a + i
  bf16x8_t pk[2][2];       // P^T of the tile before: its 32-key halves
  float m[2], l[2];        // exponent's offset; this lane's share of the sum
  float at[2];             // the offset that a tile is tried with: m, or -inf (see tile_softmax)
};

// Fragment i of a phase: i < D / 8 V's of (half st, block db), then K's of (32 dims ds, key block kb).
template <int D>
struct TileReads {
  uint32_t k[D / 32], v[D / 16];
};
template <int D>
BB_DEV u32x4_t tile_fragment(const TileReads<D>& rd, uint32_t kt, uint32_t vt, int i) {
  if (i < D / 8) {
    const int st = i / (D / 16), db = i % (D / 16);
    const uint32_t at = vt + rd.v[db] + 64 * D * st;
    const u32x2_t a = lds_tr16(at), b = lds_tr16(at + 32 * D);
    return u32x4_t{a[0], a[1], b[0], b[1]};
  }
  const int j = i - D / 8, kb = j % 4, ds = j / 4;
  return lds16(kt + rd.k[ds] + 32 * D * kb);
}
template <bool F16, int D>
BB_DEV void tile_product(TileState<D>& t, int i, bf16x8_t f) {
  if (i < D / 8) {
    const int st = i / (D / 16), db = i % (D / 16);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) t.o[db][rb] = mma16<F16>(f, t.pk[st][rb], t.o[db][rb]);
  } else {
    const int j = i - D / 8, kb = j % 4, ds = j / 4;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) t.s[kb][rb] = mma16<F16>(f, t.qf[rb][ds], ds ? t.s[kb][rb] : f32x4_t{0, 0, 0, 0});
  }
}
// Products of fragments FROM .. TO - 1, their reads kRing ahead.
template <bool F16, int D, int FROM, int TO>
BB_DEV void tile_products(TileState<D>& t, const TileReads<D>& rd, uint32_t kt, uint32_t vt) {
  constexpr int kRing = 6;
  u32x4_t ring[kRing];
#pragma unroll
  for (int i = 0; i < kRing; ++i) ring[i] = tile_fragment<D>(rd, kt, vt, FROM + i);
#pragma unroll
  for (int i = FROM; i < TO; ++i) {
    tile_product<F16, D>(t, i, as_bf16x8(ring[(i - FROM) % kRing]));
    if (i + kRing < TO) ring[(i - FROM) % kRing] = tile_fragment<D>(rd, kt, vt, i + kRing);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// P = 2^(S c - m) in 16 bits; sum: this lane's part of the row sums. (One term: its rounding is as large as the output's own;
// a second would cost half of the products again.) ROUNDED: S c is rounded before m is taken off; the asm keeps the compiler from
// fusing the two.
template <bool F16, int D, bool ROUNDED>
BB_DEV void tile_exp(TileState<D>& t, float c, const float (&m)[2], float (&sum)[2]) {
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const float nm = -m[rb];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = t.s[2 * st + e / 4][rb][e % 4];
        if constexpr (ROUNDED) {
          float x = s * c;
          asm("" : "+v"(x));
          p[e] = fast_exp2(x + nm);
        } else {
          p[e] = fast_exp2(fmaf(s, c, nm));
        }
        sum[rb] = st == 0 && e == 0 ? p[e] : sum[rb] + p[e];
      }
      t.pk[st][rb] = as_bf16x8(u32x4_t{pack2<F16>(p[0], p[1]), pack2<F16>(p[2], p[3]), pack2<F16>(p[4], p[5]), pack2<F16>(p[6], p[7])});
    }
  }
}
template <int D>
BB_DEV float tile_max(const TileState<D>& t, int rb, float c) {
  float mx = t.s[0][rb][0];
#pragma unroll
  for (int kb = 0; kb < 4; ++kb)
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, t.s[kb][rb][i]);
  return quarters_max(mx) * c;
}
template <int D>
BB_DEV void tile_rescale(TileState<D>& t, int rb, float m) {
  const float alpha = fast_exp2(t.m[rb] - m);
  t.l[rb] *= alpha;
#pragma unroll
  for (int db = 0; db < D / 16; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) t.o[db][rb][i] *= alpha;
}
// Softmax of a tile: exponentiated against the offset as it is, and again where that was too low. The exponent is the exact S c less
// m, the largest S c rounded; from 2^24 on the two lie further apart than 2, and past 2^29 no probability is left between 0 and
// infinity. So such a wave's S c are rounded too; and its tiles are tried with an offset of -inf, which is too low for all, so that
// the others pay nothing for it (a branch on a flag in each tile cost 1 to 3 %).
template <bool F16, int D>
BB_DEV void tile_softmax(TileState<D>& t, float c) {
  float sum[2];
  tile_exp<F16, D, false>(t, c, t.at, sum);
  const bool over0 = !(sum[0] <= kOver), over1 = !(sum[1] <= kOver);
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(over0 || over1) != 0, 0)) {
    float m[2];
    bool large = false;
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {
      m[rb] = fmaxf(t.m[rb], tile_max<D>(t, rb, c));
      tile_rescale<D>(t, rb, m[rb]);
      large |= m[rb] > kLowest && fabsf(m[rb]) >= 16777216.0f;
    }
    large = __builtin_amdgcn_ballot_w64(large) != 0;
    if (__builtin_expect(large, 0)) tile_exp<F16, D, true>(t, c, m, sum);
    else tile_exp<F16, D, false>(t, c, m, sum);
#pragma unroll
    for (int rb = 0; rb < 2; ++rb) {  // (in place, so that nothing is copied where this branch is not taken)
      asm("v_mov_b32 %0, %1" : "+v"(t.m[rb]) : "v"(m[rb]));
      asm("v_mov_b32 %0, %1" : "+v"(t.at[rb]) : "v"(large ? -kInf : m[rb]));
    }
  }
  t.l[0] += sum[0];
  t.l[1] += sum[1];
}

template <int D, bool F16, bool ONE>
__global__ __launch_bounds__(64 * kTileWaves, 1) void paged_tile_kernel(PagedAttnParams p) {
  using L = TileLds<D>;
  constexpr int STAGE = 2 * L::BYTES, NV = D / 8, NF = D / 4, ROW = D + 4;
  __shared__ __attribute__((aligned(1024))) uint8_t ring[kTileStages * STAGE];
  __shared__ int first[2][D];       // see first_not_finite
  __shared__ int odd[kTileStages];  // whether V's tile there may hold values that are not finite (never taken back)
  const int tid = threadIdx.x, lane = tid & 63, x = lane & 15, a = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), late = wave >> 2;  // waves w and w + 4 share a SIMD
  if (tid < kTileStages) {  // (the barrier before the first products comes before any use)
    odd[tid] = 0;
    publish();
  }
  const Item it = find_item(p, blockIdx.x, lane);
  if (it.zero) store_zeros(p, it, D, tid, 64 * kTileWaves);
  if (!it.live) return;
  const Sequence s = sequence(p.c, p.T, it.b);
  const int keys = __builtin_amdgcn_readfirstlane(pair_keys(p, s, it.tile));
  const int units = (keys + kTileRows - 1) / kTileRows;
  const int u0 = __builtin_amdgcn_readfirstlane(split_begin(units, it.splits, it.split));
  const int u1 = __builtin_amdgcn_readfirstlane(split_begin(units, it.splits, it.split + 1));
  const int begin = u0 * kTileRows, end = u1 * kTileRows < keys ? u1 * kTileRows : keys;
  const int n_tiles = (end - begin + kTileRows - 1) / kTileRows;  // 1 at least
  const int v0 = it.tile * kTileVecs;
  const int R = p.T * p.G - v0 < kTileVecs ? p.T * p.G - v0 : kTileVecs;
  const bool live = 32 * wave < R;  // a wave without vectors only loads

  // Tile i's K and V are in stage i % 4 of their halves of the ring.
  const TileLoader<D, ONE> in(p.c, it.b, it.g, end, wave, lane);
  auto k_at = [&](int i) { return ring + (i & (kTileStages - 1)) * L::BYTES; };
  auto v_at = [&](int i) { return ring + (kTileStages + (i & (kTileStages - 1))) * L::BYTES; };
  auto entries = [&](int i) { return in.entries(begin + kTileRows * i); };
  auto fetch_k = [&](int i, const typename TileLoader<D, ONE>::Entries& e) { in.load(false, k_at(i), wave, begin + kTileRows * i, e); };
  auto fetch_v = [&](int i, const typename TileLoader<D, ONE>::Entries& e) { in.load(true, v_at(i), wave, begin + kTileRows * i, e); };
  typename TileLoader<D, ONE>::Entries e0 = entries(0), e1 = entries(1), e2 = entries(2);

  // The queries' and the table's loads go out before the first tiles', which they then need not wait for.
  TileState<D> t;
  int lim[2];
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int i = 32 * wave + 16 * rb + x, v = i < R ? v0 + i : v0, j = token_of(p, v), h = it.g * p.G + v - j * p.G;
    lim[rb] = i < R ? s.seen(j) : 0;
    const uint16_t* qr = p.q + it.b * p.sq0 + h * p.sq1 + j * p.sq2 + 8 * a;
#pragma unroll
    for (int ds = 0; ds < D / 32; ++ds) t.qf[rb][ds] = as_bf16x8(ld16(qr + 32 * ds));
  }
  uint32_t most = 0;  // of the entries of the split's rows
  for (int w = (begin >> p.c.page_log2) + lane; w <= (end - 1) >> p.c.page_log2; w += 64) {
    const uint32_t e = (uint32_t)p.c.table[it.b * p.c.st + w];
    most = e > most ? e : most;
  }
  __builtin_amdgcn_sched_barrier(0);
  // Round j of loads, in the softmax of tile j, is K of tile j + 3 (over tile j - 1's, whose products the other group too is
  // past) and V of tile j + 2 (over tile j - 2's): K j + 1 and V j, wanted next, are two rounds old. At head_dim 64, where the
  // softmax is the longer phase, the round comes behind the products instead (the same tiles are free by then).
  constexpr int kRound = 2 * L::LOADS, kFlight = D == 64 ? 2 * kRound : kRound;
  fetch_k(0, e0);
  fetch_k(1, e1);
  fetch_v(0, e0);
  fetch_k(2, e2);
  fetch_v(1, e1);
  e0 = entries(3);  // of the next round's K; e2: of its V
#pragma unroll
  for (int rb = 0; rb < 2; ++rb)
#pragma unroll
    for (int ds = 0; ds < D / 32; ++ds) asm volatile("" : "+v"(t.qf[rb][ds]));  // awaited here

  // Tiles without a mask: below the rows that the tile's first token attends, if the table names a page for all of the split.
  // (What padding gets there is not stored.)
  const bool holes = __builtin_amdgcn_ballot_w64(most >= (uint32_t)p.c.pages) != 0;
  int open = __builtin_amdgcn_readfirstlane(s.seen(token_of(p, v0))) - begin;
  open = open < 0 || holes ? 0 : open / kTileRows < n_tiles ? open / kTileRows : n_tiles;

  TileReads<D> rd;
  const int vrow = 4 * a + (x >> 2);
#pragma unroll
  for (int ds = 0; ds < D / 32; ++ds) rd.k[ds] = 2 * D * x + 16 * ((4 * ds + a) ^ k_swz<D>(x));
#pragma unroll
  for (int db = 0; db < D / 16; ++db) rd.v[db] = 2 * D * vrow + 16 * ((2 * db + ((x >> 1) & 1)) ^ v_swz<D>(vrow)) + 8 * (x & 1);

  int top[2] = {-1, -1};  // a row before `lim` on a page of the table's, where tiles with a mask have one
  // The mask of tile i.
  auto mask = [&](int i) {
    const int k0 = begin + kTileRows * i;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) {
      int to = end;  // the block's rows from here on are not attended
      if (holes && (uint32_t)in.entry(k0 + 16 * kb) >= (uint32_t)p.c.pages) to = 0;
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        const int stop = to < lim[rb] ? to : lim[rb], first = k0 + 16 * kb;
        top[rb] = first < stop ? first : top[rb];
#pragma unroll
        for (int e = 0; e < 4; ++e) t.s[kb][rb][e] = first + 4 * a + e < stop ? t.s[kb][rb][e] : -kInf;
      }
    }
  };
  // A probability of 0 times a value that is not finite would be NaN. So each wave looks at the V rows that it loaded of a tile
  // that vectors attend in part, before the barrier that lets the others at them, and where one is not finite the products take
  // such values out of the operand, and vectors that attend one are NaN in that column.
  auto look_at_values = [&](int i) {
    uint32_t any = 0;
#pragma unroll
    for (int j = 0; j < L::LOADS; ++j) {
      const u32x4_t w = lds16(lds_addr(v_at(i)) + 1024 * (wave + kTileWaves * j) + 16 * lane);
#pragma unroll
      for (int e = 0; e < 4; ++e) any |= not_finite<F16>(w[e]);
    }
    if (__builtin_amdgcn_ballot_w64(any != 0)) {
      odd[i & (kTileStages - 1)] = 1;
      publish();
    }
  };
  auto odd_values = [&](int i) { return __builtin_amdgcn_readfirstlane(odd[i & (kTileStages - 1)]) != 0; };
  auto masked_values = [&](int i) {
    const uint32_t vt = lds_addr(v_at(i));
    constexpr uint32_t one = F16 ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
    for (int f = 0; f < NV; ++f) {
      const int st = f / (D / 16), db = f % (D / 16);
      int key0 = begin + kTileRows * i + 32 * st + 4 * a;
      asm volatile("" : "+v"(key0));  // (nothing of this is held across the loop around)
      u32x4_t v = tile_fragment<D>(rd, 0, vt, f), bad;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        bad[e] = not_finite<F16>(v[e]);
        v[e] &= ~bad[e];
        bad[e] &= one;
      }
      tile_product<F16, D>(t, f, as_bf16x8(v));
#pragma unroll
      for (int rb = 0; rb < 2; ++rb) {
        u32x4_t att;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + 16 * (e / 2) + 2 * (e % 2);
          att[e] = (key < lim[rb] ? one & 0xffffu : 0u) | (key + 1 < lim[rb] ? one & 0xffff0000u : 0u);
        }
        const f32x4_t hits = mma16<F16>(as_bf16x8(bad), as_bf16x8(att), f32x4_t{0, 0, 0, 0});
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (hits[e] > 0.0f) t.o[db][rb][e] = __builtin_nanf("");
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db) t.o[db][rb] = f32x4_t{0, 0, 0, 0};
    t.m[rb] = t.at[rb] = kLowest;
    t.l[rb] = 0.0f;
  }
  __builtin_amdgcn_s_waitcnt(0x0F70 | 2 * kRound);  // K of tile 0 has landed
  ring_barrier();
  if (late) ring_barrier();  // the second group runs one phase behind
  auto round = [&](int j) {
    fetch_k(j + 3, e0);
    fetch_v(j + 2, e2);
    e2 = e0;
    e0 = entries(j + 4);
  };
  if (live) tile_products<F16, D, NV, NF>(t, rd, lds_addr(k_at(0)), 0);
  if (D == 64) round(0);
  __builtin_amdgcn_s_waitcnt(0x0F70 | kFlight);
  if (open == 0) look_at_values(0);
  ring_barrier();
  if (live) {
    if (open == 0) mask(0);
    tile_softmax<F16, D>(t, p.scale);
  }
  if (D != 64) round(0);
  ring_barrier();
  for (int i = 1; i < open; ++i) {
    __builtin_amdgcn_s_setprio(1);
    if (live) tile_products<F16, D, 0, NF>(t, rd, lds_addr(k_at(i)), lds_addr(v_at(i - 1)));
    if (D == 64) round(i);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_s_waitcnt(0x0F70 | kFlight);
    ring_barrier();
    if (live) tile_softmax<F16, D>(t, p.scale);
    if (D != 64) round(i);
    ring_barrier();
  }
  auto values = [&](int i) {
    if (i >= open && odd_values(i)) masked_values(i);
    else tile_products<F16, D, 0, NV>(t, rd, 0, lds_addr(v_at(i)));
  };
#pragma unroll 1
  for (int i = open > 1 ? open : 1; i < n_tiles; ++i) {
    if (live) {
      values(i - 1);
      tile_products<F16, D, NV, NF>(t, rd, lds_addr(k_at(i)), 0);
    }
    if (D == 64) round(i);
    __builtin_amdgcn_s_waitcnt(0x0F70 | kFlight);
    look_at_values(i);
    ring_barrier();
    if (live) {
      mask(i);
      tile_softmax<F16, D>(t, p.scale);
    }
    if (D != 64) round(i);
    ring_barrier();
  }
  if (live) values(n_tiles - 1);
  if (!late) ring_barrier();  // the groups meet again
  __builtin_amdgcn_s_waitcnt(0x0F70);  // nothing lands in LDS any more
  bool bad[2];  // sums that are not finite
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    t.l[rb] = quarters_sum(t.l[rb]);
    f32x4_t size = {0, 0, 0, 0};
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
#pragma unroll
      for (int e = 0; e < 4; ++e) size[e] += fabsf(t.o[db][rb][e]);
    bad[rb] = lim[rb] > 0 && t.l[rb] > 0.0f && t.l[rb] < kInf && !(size[0] + size[1] + size[2] + size[3] < kInf);
  }
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad[0] || bad[1]) != 0, 0)) {
    constexpr int N = D / 64;
    int pos[N], neg[N];
    first_not_finite<F16>(p.c, it.b, in.vh, begin, end, N * lane, pos, neg);
#pragma unroll
    for (int k = 0; k < N; ++k) {  // (the same from every wave that comes here)
      first[0][N * lane + k] = pos[k];
      first[1][N * lane + k] = neg[k];
    }
    publish();
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
      if (bad[rb])
#pragma unroll
        for (int db = 0; db < D / 16; ++db)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            t.o[db][rb][e] = with_infinities(t.o[db][rb][e], first[0][16 * db + 4 * a + e], first[1][16 * db + 4 * a + e], lim[rb]);
  }
#pragma unroll
  for (int rb = 0; rb < 2; ++rb) {
    const int i = 32 * wave + 16 * rb + x;
    const float l = t.l[rb];
    const bool seen = lim[rb] > 0 && (open > 0 || top[rb] >= 0);
    const float inv = 1.0f / l;  // (another rounding of 2^-24, instead of 64 divisions a lane)
    if (i >= R) continue;
    if (it.splits == 1) {
      const int v = v0 + i, j = token_of(p, v), h = it.g * p.G + v - j * p.G;
      uint16_t* to = p.out + it.b * p.so0 + h * p.so1 + j * p.so2 + 4 * a;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) {
        f32x4_t o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = seen ? t.o[db][rb][e] * inv : 0.0f;
        *reinterpret_cast<u32x2_t*>(to + 16 * db) = u32x2_t{pack2<F16>(o[0], o[1]), pack2<F16>(o[2], o[3])};
      }
    } else {
      float* to = p.part + ((int64_t)it.slot * kTileVecs + i) * ROW;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) *reinterpret_cast<f32x4_t*>(to + 16 * db + 4 * a) = t.o[db][rb];
      if (a == 0) {
        to[D] = seen ? t.m[rb] : -kInf;
        to[D + 1] = l;
      }
    }
  }
}

// The splits' states of each vector under one maximum. Split s of n of a pair merges, in gridDim.y workgroups, the s-th part of
// its vectors: a group of D / 4 lanes a vector, or all groups of the workgroup one vector where that is its part. 4 us traced, of
// which 2 lie beside the attention's end, whatever it merges; a quarter or half of the workgroups in a loop over the slots are no
// faster.
template <int D, bool F16>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(PagedAttnParams p) {
  constexpr int LPV = D / 4, NG = kThreads / LPV, ROW = D + 4;
  __shared__ float st[NG][ROW];
  const int tid = threadIdx.x, grp = tid / LPV, d = 4 * (tid % LPV);
  const int4 rec = p.plan[blockIdx.x];
  if ((int)blockIdx.x >= p.plan[p.slots].x) return;
  const int b = rec.x, tile = rec.y, g = rec.z, split = rec.w & 0xffff, splits = rec.w >> 16;
  const int R = p.T * p.G - tile * p.VT < p.VT ? p.T * p.G - tile * p.VT : p.VT;
  const int parts = splits * gridDim.y, part = split * gridDim.y + blockIdx.y;
  const int from = R * part / parts, to = R * (part + 1) / parts;
  const float* slots = p.part + (int64_t)(blockIdx.x - split) * p.VT * ROW;
  float M, L;
  f32x4_t O;
  auto merge = [&](int v, int first, int step) {  // splits first, first + step, ..
    const float* src = slots + (int64_t)v * ROW;
    constexpr int U = 4;  // whose loads are in flight together
    M = -kInf;
    L = 0.0f;
    O = f32x4_t{0, 0, 0, 0};
    for (int i = first; i < splits; i += U * step) {
      float m[U], l[U], mn = M;
      f32x4_t t[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int at = i + k * step < splits ? i + k * step : i;
        const float* f = src + (int64_t)at * p.VT * ROW;
        const u32x2_t ml = *reinterpret_cast<const u32x2_t*>(f + D);
        m[k] = __uint_as_float(ml[0]);
        l[k] = __uint_as_float(ml[1]);
        t[k] = *reinterpret_cast<const f32x4_t*>(f + d);
      }
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (i + k * step >= splits) m[k] = -kInf;
        mn = fmaxf(mn, m[k]);
      }
      const float off = mn == -kInf ? 0.0f : mn, was = fast_exp2(M - off);
      M = mn;
      L *= was;
#pragma unroll
      for (int j = 0; j < 4; ++j) O[j] *= was;
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (i + k * step >= splits) continue;
        const float wt = fast_exp2(m[k] - off);
        L = fmaf(wt, l[k], L);
#pragma unroll
        for (int j = 0; j < 4; ++j) O[j] = fmaf(wt, t[k][j], O[j]);
      }
    }
  };
  // Infinities are attended values (see first_not_finite), which a weight of 0 does not make NaN.
  auto look_up = [&](int v) {
    if (fabsf(O[0]) + fabsf(O[1]) + fabsf(O[2]) + fabsf(O[3]) < kInf || !(L > 0.0f && L < kInf)) return;
    f32x4_t sum = {0, 0, 0, 0};
    for (int i = 0; i < splits; ++i) {
      const f32x4_t o = *reinterpret_cast<const f32x4_t*>(slots + ((int64_t)i * p.VT + v) * ROW + d);
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += fabsf(o[j]) < kInf ? 0.0f : o[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) O[j] = sum[j] == 0.0f ? O[j] : sum[j];
  };
  if (to - from > 1) {
    for (int v = from + grp; v < to; v += NG) {
      merge(v, 0, 1);
      look_up(v);
      store_output<F16>(p, b, g, tile * p.VT + v, d, O, M, L);
    }
    return;
  }
  if (to == from) return;
  merge(from, grp, NG);
  *reinterpret_cast<f32x4_t*>(&st[grp][d]) = O;
  if (d == 0) {
    st[grp][D] = M;
    st[grp][D + 1] = L;
  }
  __syncthreads();
  if (grp != 0) return;
  M = -kInf;
#pragma unroll
  for (int i = 0; i < NG; ++i) M = fmaxf(M, st[i][D]);
  const float off = M == -kInf ? 0.0f : M;
  L = 0.0f;
  O = f32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    const float wt = fast_exp2(st[i][D] - off);
    L = fmaf(wt, st[i][D + 1], L);
#pragma unroll
    for (int k = 0; k < 4; ++k) O[k] = fmaf(wt, st[i][d + k], O[k]);
  }
  look_up(from);
  store_output<F16>(p, b, g, tile * p.VT + from, d, O, M, L);
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t stream) {
  const int64_t units = (int64_t)p.B * p.T * (p.H + 2 * p.Hkv), per = kThreads / (p.D / 16);
  const dim3 grid((unsigned)((units + per - 1) / per));
  if (p.D == 128) {
    if (p.f16) paged_append_kernel<128, true><<<grid, kThreads, 0, stream>>>(p);
    else paged_append_kernel<128, false><<<grid, kThreads, 0, stream>>>(p);
  } else {
    if (p.f16) paged_append_kernel<64, true><<<grid, kThreads, 0, stream>>>(p);
    else paged_append_kernel<64, false><<<grid, kThreads, 0, stream>>>(p);
  }
  return hipGetLastError();
}

namespace {
template <int D, bool F16, int NR>
hipError_t attend(const PagedAttnParams& p, hipStream_t stream) {
  if constexpr (NR == 0) {
    if (1 << p.c.page_log2 >= kTileRows) paged_tile_kernel<D, F16, true><<<p.grid, 64 * kTileWaves, 0, stream>>>(p);
    else paged_tile_kernel<D, F16, false><<<p.grid, 64 * kTileWaves, 0, stream>>>(p);
  }
  else if (NR == 2 && p.tiles > 1) paged_attn_kernel<D, F16, 2, true, 0><<<p.grid, kThreads, 0, stream>>>(p);  // (a step)
  else if (p.knew) paged_attn_kernel<D, F16, NR, true, 2><<<p.grid, kThreads, 0, stream>>>(p);
  else paged_attn_kernel<D, F16, NR, false, 2><<<p.grid, kThreads, 0, stream>>>(p);
  if (p.part) {
    const dim3 grid(p.slots, p.VT > 32 ? 4 : 1);  // a tile's parts are many vectors
    paged_merge_kernel<D, F16><<<grid, kThreads, 0, stream>>>(p);
  }
  return hipGetLastError();
}
template <int D, bool F16>
hipError_t attend(const PagedAttnParams& p, hipStream_t stream) {
  if (p.VT == 16) return attend<D, F16, 1>(p, stream);
  if (p.VT == 32) return attend<D, F16, 2>(p, stream);
  return attend<D, F16, 0>(p, stream);
}
}  // namespace

hipError_t launch_paged_attention(const PagedAttnParams& p, hipStream_t stream) {
  if (p.items) paged_plan_kernel<<<1, kPlanThreads, 0, stream>>>(p);
  if (p.D == 128) return p.f16 ? attend<128, true>(p, stream) : attend<128, false>(p, stream);
  return p.f16 ? attend<64, true>(p, stream) : attend<64, false>(p, stream);
}

}  // namespace bb
