// KV cache in 4 bits: the write, the read back, and the exact attention of a few query tokens over the packed rows.
//
// A row of D elements is D / 32 groups of 32. Per group, with min and max clamped to +-65504 and NaN left out of them:
//   z = fp16(min), s = fp16(max((max - z) / 15, 0)), code = rint((x - z) / s) clamped to 0..15 (0 where s = 0 or x is NaN),
// each operation in fp32; the value is s * code + z in fp32 (s * code is exact). A group of NaN alone has s = z = 0. s and z
// are rounded before the codes are taken, so the codes make up for their rounding. Byte b of a packed row holds elements 2 b
// (low four bits) and 2 b + 1.
//
// The cache is head-major, codes [Hkv, cap, D / 2] and params [Hkv, cap, D / 32] of (s, z): the rows of one KV head are
// one contiguous range, so that a workgroup that streams them reads whole 128-byte lines (64-byte rows of one head between
// those of the others would leave half of every line to another workgroup).
#include "bb_common.h"
#include "bb_internal.h"
#include "bb_slots.h"

namespace bb {
namespace {

constexpr int kKindBf16 = 0, kKindF32 = 1, kKindF16 = 2;
constexpr int kGroup = 32;  // elements that share a (scale, minimum)
constexpr float kF16Max = 65504.0f;

BB_DEV float f16_lo(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w & 0xffffu)); }
BB_DEV float f16_hi(uint32_t w) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(w >> 16)); }
// f rounded to nearest even. f passes through an empty asm: the compiler would otherwise shrink an fp32 operation before it to one
// that rounds to fp16 directly, where the format rounds to fp32 first.
BB_DEV uint32_t f16_bits(float f) {
  asm("" : "+v"(f));
  return __builtin_bit_cast(uint16_t, (_Float16)f);
}

// N (a multiple of 8) elements of a row at x (16-byte aligned), in fp32.
template <int KIND, int N>
BB_DEV void load_row(const void* x, int64_t off, float (&v)[N]) {
  if constexpr (KIND == kKindF32) {
    const f32x4_t* p = reinterpret_cast<const f32x4_t*>(reinterpret_cast<const float*>(x) + off);
#pragma unroll
    for (int j = 0; j < N / 4; ++j) {
      const f32x4_t a = p[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[4 * j + i] = a[i];
    }
  } else {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(x) + off;
#pragma unroll
    for (int j = 0; j < N / 8; ++j) {
      const u32x4_t a = ld16(p + 8 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[8 * j + 2 * i] = KIND == kKindF16 ? f16_lo(a[i]) : __uint_as_float(a[i] << 16);
        v[8 * j + 2 * i + 1] = KIND == kKindF16 ? f16_hi(a[i]) : __uint_as_float(a[i] & 0xffff0000u);
      }
    }
  }
}

// Quantises the N elements v of a lane (8 or 16; the 32 / N lanes of a group are neighbours and all take part): their codes,
// little-endian, and the group's (s, z) as packed fp16.
//   * (max - z) / 15 is the correctly rounded quotient: one step of Newton's iteration on the residual, which an fma gives
//     exactly, with the correctly rounded reciprocal of 15.
//   * (x - z) / s likewise, with the hardware's reciprocal: off the correctly rounded quotient at most where that is far from
//     a half (tried for every fp16 s, reciprocals off by up to 2 ulps and 40 floats to each side of every half).
// v holds infinities and values past fp16's range until the rare branch puts them in it (the residual of an infinity is NaN).
template <int N>
BB_DEV void quant_4bit(float (&v)[N], uint32_t (&w)[N / 8], uint32_t& param) {
  float lo = __builtin_huge_valf(), hi = -__builtin_huge_valf();
#pragma unroll
  for (int i = 0; i < N; ++i) {  // NaN operands are passed over
    lo = fminf(lo, v[i]);
    hi = fmaxf(hi, v[i]);
  }
  lo = fminf(lo, dpp_mov<0xB1>(lo));
  hi = fmaxf(hi, dpp_mov<0xB1>(hi));
  if constexpr (N == 8) {
    lo = fminf(lo, dpp_mov<0x4E>(lo));
    hi = fmaxf(hi, dpp_mov<0x4E>(hi));
  }
  const bool some = lo <= hi;
  if (hi > kF16Max) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] > kF16Max ? kF16Max : v[i];
  }
  lo = some ? fminf(fmaxf(lo, -kF16Max), kF16Max) : 0.0f;
  hi = some ? fminf(fmaxf(hi, -kF16Max), kF16Max) : 0.0f;
  const uint32_t zb = f16_bits(lo);
  const float z = f16_lo(zb);
  const float range = fmaxf(hi - z, 0.0f), q15 = range * (1.0f / 15.0f);
  const uint32_t sb = f16_bits(fmaf(fmaf(-15.0f, q15, range), 1.0f / 15.0f, q15));
  const float s = f16_lo(sb);
  param = sb | (zb << 16);
  const float inv = s > 0.0f ? __builtin_amdgcn_rcpf(s) : 0.0f;
#pragma unroll
  for (int j = 0; j < N / 8; ++j) {
    float part[2] = {0.0f, 0.0f};  // four codes each, exact in fp32
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = v[8 * j + i] - z, t = d * inv, c = rintf(fmaf(fmaf(-t, s, d), inv, t));
      // (NaN comes out of the median as 0)
      part[i / 4] = fmaf(__builtin_amdgcn_fmed3f(c, 0.0f, 15.0f), (float)(1 << (4 * (i % 4))), part[i / 4]);
    }
    w[j] = (uint32_t)part[0] | ((uint32_t)part[1] << 16);
  }
}

struct Int4Set {  // one tensor's rows and their place in the cache
  const void* x;
  uint8_t* q;
  uint32_t* p;
  int64_t sx0, sx1;  // head and row stride of x (elements)
  int64_t sq0, sp0;  // head strides of q (bytes) and p (groups)
};

// A lane takes half a group (16 elements) of a row; blockIdx.x counts heads within blocks of rows, so that the rows of a
// token's heads, which neighbour each other where a projection left them, are read at about the same time; blockIdx.y is the
// tensor (K, V). Bound by memory: K and V of 131072 rows x 8 heads x 128 in bf16 (0.54 GB read, 0.17 GB written) take 123 us,
// 5.7 TB/s; with true divisions, 8 elements a lane, the arithmetic set the time (208 us).
template <int D, int KIND>
__global__ __launch_bounds__(256) void int4_quantize_kernel(Int4Set s0, Int4Set s1, int heads, int64_t rows) {
  const Int4Set& s = blockIdx.y ? s1 : s0;
  constexpr int LPR = D / 16;
  const int h = blockIdx.x % (unsigned)heads, c = threadIdx.x % LPR;
  const int64_t row = (int64_t)(blockIdx.x / (unsigned)heads) * (256 / LPR) + threadIdx.x / LPR;
  if (row >= rows) return;  // the lanes of a row leave together
  float v[16];
  load_row<KIND>(s.x, h * s.sx0 + row * s.sx1 + 16 * c, v);
  uint32_t param, w[2];
  quant_4bit(v, w, param);
  *reinterpret_cast<u32x2_t*>(s.q + h * s.sq0 + row * (D / 2) + 8 * c) = u32x2_t{w[0], w[1]};
  if (c % 2 == 0) s.p[h * s.sp0 + row * (D / kGroup) + c / 2] = param;
}

struct Int4ReadSet {
  const uint8_t* q;
  const uint32_t* p;
  void* out;  // [heads, rows, D] contiguous
  int64_t sq0, sp0;
};

// A lane takes 8 elements; memory alone bounds it (131072 rows as above: 0.70 GB in 138 us, 5.1 TB/s, where a copy reaches 4.9).
// The values are stored past the caches (the stores are as fast, and packed rows that lie in the 256 MB cache stay there: K and V
// of 65536 rows x 8 heads x 128 read back 74 -> 48 us, of 131072 rows 145 -> 140; reading the values next is no slower: at
// 16 MB of them 10.8 -> 10.6 us for both, at 64 MB 28.6 -> 26.1).
template <int D>
__global__ __launch_bounds__(256) void int4_dequantize_kernel(Int4ReadSet s0, Int4ReadSet s1, int kind, int64_t rows) {
  const Int4ReadSet& s = blockIdx.z ? s1 : s0;
  constexpr int LPR = D / 8;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR, h = blockIdx.y;
  if (row >= rows) return;
  const uint32_t w = *reinterpret_cast<const uint32_t*>(s.q + h * s.sq0 + row * (D / 2) + 4 * c);
  const uint32_t pr = s.p[h * s.sp0 + row * (D / kGroup) + c / 4];
  const float sc = f16_lo(pr), z = f16_hi(pr);
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = fmaf(sc, (float)((w >> (4 * i)) & 15u), z);
  const int64_t off = (h * rows + row) * D + 8 * c;
  if (kind == kKindF32) {
    f32x4_t* o = reinterpret_cast<f32x4_t*>(reinterpret_cast<float*>(s.out) + off);
    __builtin_nontemporal_store(f32x4_t{v[0], v[1], v[2], v[3]}, o);
    __builtin_nontemporal_store(f32x4_t{v[4], v[5], v[6], v[7]}, o + 1);
  } else {
    u32x4_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = kind == kKindF16 ? f16_bits(v[2 * i]) | (f16_bits(v[2 * i + 1]) << 16) : pack2<false>(v[2 * i], v[2 * i + 1]);
    __builtin_nontemporal_store(o, reinterpret_cast<u32x4_t*>(reinterpret_cast<uint16_t*>(s.out) + off));
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Attention over the packed rows, split over the keys. Workgroup (split, KV head, pass): 4 waves against the split's keys,
// wave w taking chunks w, w + 4, ... of 64 keys (128 at head_dim 64). The query vectors of a KV head are its T tokens x G
// heads, token-major: up to 4 go to int4_decode_kernel, more to int4_decode_wide_kernel in passes of 16. The length may come
// from device memory; every launch shape depends on host values alone.
//
// Mathematics. With k = s c + z per group of 32 (c the codes), q.k = sum_g s_g (q_g . c_g) + z_g sum(q_g), and
// o = sum_j p_j s_j c_j + sum_j p_j z_j per column group: the codes go to the matrix cores as they are, exact in 16 bits, and
// scales and minima are applied in fp32 to the sums (scores) or to the probabilities (values). In the scores a code becomes a
// 16-bit float base + c by an and-or per two codes (see Codes), and the bases are taken back from the sums; in the values it is
// a subnormal number (see ValueCodes).
//
// A chunk's 10 KB (codes and params of K and of V) stream straight into the wave's LDS with ten buffer loads that cover
// whole lines, two chunks ahead. Pieces land so that the operand reads meet no bank twice: see the offsets at each. V rows
// are transposed on the way to the matrix cores by ds_read_b64_tr_b4 (a lane gets 16 keys of one column).
constexpr int kVecs = 16;            // query vectors of a pass of the wide kernel
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kStage = 10240;        // K codes 4096 | K params 1024 | V codes 4096 | V params 1024
constexpr int kKp = 4096, kVq = 5120, kVp = 9216;
constexpr float kOver = 256.0f;      // a probability past this moves the running maximum
constexpr float kLowest = -3.402823466e38f;  // -FLT_MAX, what a running maximum starts from: no finite score lies below it

typedef int v2i_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

BB_DEV int64_t live_length(const Int4DecodeParams& p, int64_t raw) { return raw < 0 ? 0 : raw > p.cap ? p.cap : raw; }
// Keys of a split: the live length in equal parts of whole 16 keys (the bytes per CU set the time, so the parts are not
// rounded to chunks); the host passes it as p.len unless the length is in device memory. ceil(n / n_splits) from the rounded
// reciprocal, put right by one where it is off: a 64-bit division is hundreds of instructions ahead of the first load.
BB_DEV int64_t split_keys(const Int4DecodeParams& p, int64_t n) {
  int64_t len = (int64_t)((double)n * p.inv_splits);
  if (len * p.n_splits < n) ++len;
  len = (len + 15) & ~(int64_t)15;
  return len < kInt4MinSplit ? kInt4MinSplit : len;
}
// The token of query vector v (v / G; v < 2^20, so the product with the rounded reciprocal is off by less than 1 / (2 G)).
BB_DEV int token_of(const Int4DecodeParams& p, int v) { return (int)(((float)v + 0.5f) * p.inv_G); }

// The first keys that token t attends of a cache of n rows; none or less: the token's output is zeros. Every other one is the
// quotient of its sums, so that a query that is not finite, and scores that are all -inf, give NaN as the formula does.
BB_DEV int64_t attended(const Int4DecodeParams& p, int64_t n, int t) { return p.causal ? n - p.T + 1 + t : n; }

BB_DEV f32x4_t mma16_bf16(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
template <bool F16>
BB_DEV f32x4_t mma16(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                  0);
  else return mma16_bf16(a, b, c);
}

// Eight K codes as 16-bit floats base + c, in the order 0, 4, 1, 5, 2, 6, 3, 7 (the halves of the word side by side). In fp16
// 64.0 has an ulp of 1/16: bits 4..7 of a half are a code in its place. In bf16 128.0 has an ulp of 1 (bits 0..3) and 16.0 one
// of 1/8 (bits 3..6); no place serves two pairs. So of the four pairs three take a shift. The constants stay in registers
// (masks scalar, bases vector), where one v_and_or_b32 takes both; as literals they cost an instruction more.
template <bool F16>
struct Codes {
  uint32_t mask0, mask, base0, base;
  BB_DEV Codes()
      : mask0(0x000f000fu), mask(F16 ? 0x00f000f0u : 0x00780078u), base0(0x43004300u), base(F16 ? 0x54005400u : 0x41804180u) {
    asm("" : "+s"(mask));
    asm("" : "+v"(base));
    if constexpr (!F16) {
      asm("" : "+s"(mask0));
      asm("" : "+v"(base0));
    }
  }
  BB_DEV bf16x8_t operator()(uint32_t w) const {
    if constexpr (F16)
      return as_bf16x8(u32x4_t{((w << 4) & mask) | base, (w & mask) | base, ((w >> 4) & mask) | base, ((w >> 8) & mask) | base});
    else
      return as_bf16x8(u32x4_t{(w & mask0) | base0, ((w >> 1) & mask) | base, ((w >> 5) & mask) | base, ((w >> 9) & mask) | base});
  }
  // A fragment of the bases themselves.
  BB_DEV static bf16x8_t bases() {
    if constexpr (F16) return as_bf16x8(u32x4_t{0x54005400u, 0x54005400u, 0x54005400u, 0x54005400u});
    else return as_bf16x8(u32x4_t{0x43004300u, 0x41804180u, 0x41804180u, 0x41804180u});
  }
};

// Eight V codes as subnormal bf16 numbers, in the same order: the matrix cores take them exactly, and no base has to come off
// again. (With bases the sums are 17 times what is wanted, and so is their rounding: over 131072 rows 3.6e-5 of an output's norm
// instead of 6e-6, over 1000000 in 64 splits 2.7e-4 instead of 4e-5, at the same time.) Bits 0..3 of a half are c * 2^-133, bits
// 3..6 c * 2^-130; the first pair's probabilities carry the factor of 8 between them (prob_up). 2^64 on all of them keeps the
// products in fp32's normal range.
struct ValueCodes {
  uint32_t mask0, mask;
  BB_DEV ValueCodes() : mask0(0x000f000fu), mask(0x00780078u) {}
  BB_DEV bf16x8_t operator()(uint32_t w) const {
    return as_bf16x8(u32x4_t{w & mask0, (w >> 1) & mask, (w >> 5) & mask, (w >> 9) & mask});
  }
};
BB_DEV float prob_up(bool first_pair) { return first_pair ? 0x1p67f : 0x1p64f; }
constexpr float kSumDown = 0x1p66f;  // what brings the sums back: 2^130 / 2^64

// a times the low / high fp16 half of w, in one instruction (fp32 product, rounded once).
BB_DEV float mul_lo(float a, uint32_t w) {
  float r;
  asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel_hi:[0,1,0]" : "=v"(r) : "v"(a), "v"(w));
  return r;
}
BB_DEV float mul_hi(float a, uint32_t w) {
  float r;
  asm("v_fma_mix_f32 %0, %1, %2, 0 op_sel:[0,1,0] op_sel_hi:[0,1,0]" : "=v"(r) : "v"(a), "v"(w));
  return r;
}

// The largest / sum over the 16 lanes of a DPP row, in every lane.
BB_DEV float row_max(float v) {
  v = fmaxf(v, dpp_mov<0x128>(v));
  v = fmaxf(v, dpp_mov<0x124>(v));
  v = fmaxf(v, dpp_mov<0x122>(v));
  return fmaxf(v, dpp_mov<0x121>(v));
}
BB_DEV float row_sum(float v) {
  v += dpp_mov<0x128>(v);
  v += dpp_mov<0x124>(v);
  v += dpp_mov<0x122>(v);
  return v + dpp_mov<0x121>(v);
}
// Rows 0, 2 of the result: a summed over the row pair (0, 1), (2, 3); rows 1, 3: b.
BB_DEV float sum_rows16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Lanes 0..31: a summed over the wave's halves; lanes 32..63: b.
BB_DEV float sum_rows32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The sum / largest over the four quarters of the wave, in every lane.
BB_DEV float quarters_sum(float v) { return xhalf_sum(sum_rows16(v, v)); }
BB_DEV float quarters_max(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return xhalf_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
BB_DEV float lane_value(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// LDS written by this wave before is what it reads after (LDS operations of one wave run in order: this orders the compiler).
BB_DEV void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Eight bytes of LDS per lane, transposed in 4-bit units: lane l of 16 gets column l of the 16 lanes' rows, row r in four-bit
// place r. `restrict` tells the compiler that no load into LDS in flight writes what is read here (the loop waits for the
// chunk itself); without it the compiler waits for every load in flight, the next chunk's too.
BB_DEV v2i_t read_tr4(const uint8_t* __restrict__ at) {
  return __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) v2i_t*)at);
}

// Where a chunk's rows lie in its stage; key (0 .. CH - 1) is the row's place in the chunk. In a region of 16 rows K row
// b3 b2 b1 b0 is at b2 b0 b3 b1, so that the 16 lanes of a score step, whose rows differ in b3, b1 and the region, read
// 16-byte pieces in every bank once (the regions' pieces are shifted against each other as well).
BB_DEV int k_place(int row) { return ((row >> 2) & 1) << 3 | (row & 1) << 2 | ((row >> 3) & 1) << 1 | ((row >> 1) & 1); }
BB_DEV int k_unplace(int pos) { return ((pos >> 1) & 1) << 3 | (pos >> 3) << 2 | (pos & 1) << 1 | ((pos >> 2) & 1); }
template <int D>
BB_DEV int k_code_at(int key, int piece) {
  const int region = (key >> 4) & 3, pos = k_place(key & 15);
  if constexpr (D == 128) return 1024 * region + 64 * pos + 16 * (piece ^ (-region & 3));
  else return 2048 * (key >> 6) + 512 * region + 32 * (pos ^ (4 * (region >> 1))) + 16 * piece;
}
// V row r's piece is shifted by the row, so that 16 rows' reads of one column block meet no bank twice.
template <int D>
BB_DEV int v_code_at(int key, int piece) {
  const int region = (key >> 4) & 3, row = key & 15;
  if constexpr (D == 128) return 1024 * region + 64 * row + 16 * (piece ^ (row >> 2));
  else return 2048 * (key >> 6) + 512 * region + 32 * row + 16 * (piece ^ (row >> 3));
}
// Where lane (k, a) points for columns 16 db .. 16 db + 15 of the 64 keys of half hv: row 16 a + k, 8 bytes.
template <int D>
BB_DEV int v_block_at(int k, int a, int hv, int db) {
  if constexpr (D == 128) return 1024 * a + 64 * k + 16 * ((db >> 1) ^ (k >> 2)) + 8 * (db & 1);
  else return 2048 * hv + 512 * a + 32 * k + 16 * ((db >> 1) ^ (k >> 3)) + 8 * (db & 1);
}
// A key's params: 16 u + k of lane k and score step u; at head_dim 64 two neighbouring keys share a 16-byte piece.
template <int D>
BB_DEV int param_at(int key) {
  const int k = 4 * ((key >> 4) & 3) + 2 * ((key >> 3) & 1) + ((key >> 1) & 1), u = (key >> 2) & 1, odd = key & 1;
  if constexpr (D == 128) return 16 * (16 * (u + 2 * odd) + k);
  else return 512 * u + 256 * (key >> 6) + 16 * k + 8 * odd;
}

// The step's new rows among the keys [first, first + CH) of the split (fewer than `count`): quantised into the chunk in
// LDS, over what the cache held there, and by the first pass into the cache. No other chunk holds them, so nothing waits
// for the stores.
template <int D, bool F16, int CH>
BB_DEV void append_rows(const Int4DecodeParams& p, int64_t raw, int64_t begin, int first, int count, int g, int lane,
                        uint8_t* s) {
  constexpr int LPR = D / 8;
  const int c = lane % LPR;
  for (int i = lane / LPR; i < 2 * p.T; i += 64 / LPR) {  // the lanes of a row stay together
    const int t = i >> 1, vt = i & 1;
    const int64_t row = raw - p.T + t, at = row - begin;
    if (at < first || at >= first + CH || at >= count) continue;
    float v[8];
    load_row<F16 ? kKindF16 : kKindBf16>(vt ? p.vnew : p.knew,
                                         vt ? g * p.svn0 + t * p.svn1 + 8 * c : g * p.skn0 + t * p.skn1 + 8 * c, v);
    uint32_t param, codes[1];
    quant_4bit(v, codes, param);
    const uint32_t w = codes[0];
    const int key = (int)at - first;
    *reinterpret_cast<uint32_t*>(s + (vt ? kVq + v_code_at<D>(key, c / 4) : k_code_at<D>(key, c / 4)) + 4 * (c % 4)) = w;
    if (c % 4 == 0) *reinterpret_cast<uint32_t*>(s + (vt ? kVp : kKp) + param_at<D>(key) + c) = param;
    if (blockIdx.z == 0) {
      *reinterpret_cast<uint32_t*>((vt ? p.vq + g * p.svq : p.kq + g * p.skq) + row * (D / 2) + 4 * c) = w;
      if (c % 4 == 0) (vt ? p.vp + g * p.svp : p.kp + g * p.skp)[row * (D / kGroup) + c / 4] = param;
    }
  }
}

// One wave's stream of chunks: where lane l's 16 bytes of each load come from (load i lands at 1024 i + 16 l). Loads cover
// whole contiguous kilobytes; inside, pieces are placed for the reads. Lane k of a score step u works on
//   key(k, u) = 16 (k >> 2) + 8 ((k >> 1) & 1) + 4 (u & 1) + 2 (k & 1) + (u >> 1)     (+ 64 in the second half of 128)
// so that a lane's four steps are four neighbouring elements of the value operand (the codes' order).
BB_DEV int key_of_lane(int k) { return 16 * (k >> 2) + 8 * ((k >> 1) & 1) + 2 * (k & 1); }
BB_DEV int key_of_step(int u) { return 4 * (u & 1) + (u >> 1); }
template <int D>
struct Stream {
  uint32_t koff[2], voff, poff;
  const uint8_t *kq, *vq;
  const uint32_t *kp, *vp;
  int count;
  BB_DEV Stream(const Int4DecodeParams& p, int g, int64_t begin, int count_, int lane) : count(count_) {
    const int k = lane & 15;
    if constexpr (D == 128) {
      koff[0] = koff[1] = 64 * k_unplace(lane >> 2) + 16 * (lane & 3);  // load i: pieces xor -i & 3
      voff = 64 * (lane >> 2) + 16 * ((lane & 3) ^ (lane >> 4));
      poff = 16 * (key_of_lane(k) + key_of_step(lane >> 4));
    } else {
      const int pos = (lane >> 1) & 15;
      koff[0] = 512 * (lane >> 5) + 32 * k_unplace(pos) + 16 * (lane & 1);
      koff[1] = 512 * (lane >> 5) + 32 * k_unplace(pos ^ 4) + 16 * (lane & 1);  // odd loads: regions 2 and 3
      voff = 512 * (lane >> 5) + 32 * pos + 16 * ((lane & 1) ^ (pos >> 3));
      poff = 8 * (64 * ((lane >> 4) & 1) + key_of_lane(k) + 4 * (lane >> 5));
    }
    kq = p.kq + g * p.skq + begin * (D / 2);
    vq = p.vq + g * p.svq + begin * (D / 2);
    kp = p.kp + g * p.skp + begin * (D / kGroup);
    vp = p.vp + g * p.svp + begin * (D / kGroup);
  }
  // Chunk c's K or V into `stage`: always five loads, so that the counts the waits go by are exact; past the split's last chunk
  // they read nothing (the buffers' ranges end with it) and land zeros.
  BB_DEV void fetch_k(uint8_t* stage, int c) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t off = D == 128 ? koff[0] ^ (16 * (-i & 3)) : koff[i & 1];  // head_dim 128: bits 4 and 5 are the piece
      load(kq, D / 2, stage + 1024 * i, c * 4096 + 1024 * i + off);
    }
    load(kp, D / 8, stage + kKp, c * 1024 + poff);
  }
  BB_DEV void fetch_v(uint8_t* stage, int c) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) load(vq, D / 2, stage + kVq + 1024 * i, c * 4096 + 1024 * i + voff);
    load(vp, D / 8, stage + kVp, c * 1024 + poff);
  }
  BB_DEV void load(const void* base, int row_bytes, uint8_t* to, uint32_t off) const {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, count * row_bytes, 0x00020000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, reinterpret_cast<lds_void*>(reinterpret_cast<uintptr_t>(to)), 16, off, 0, 0,
                                             2 /* non-temporal */);
  }
};

// A split's part of a call.
struct Part {
  int64_t n, raw, begin;  // length, length before clamping, first key
  int count, new_first;   // keys, and the first of them that may be a new row
  BB_DEV Part(const Int4DecodeParams& p, int split) {
    raw = n = p.n;
    int64_t len = p.len;
    if (p.n_dev) {
      raw = *p.n_dev;
      n = live_length(p, raw);
      len = split_keys(p, n);
    }
    begin = split * len;
    const int64_t left = n - begin;
    count = (int)(left < 0 ? 0 : left < len ? left : len);
    // the length before clamping places the new rows; those that it puts outside the cache are left out
    const int64_t at = raw - p.T - begin;
    new_first = p.knew != nullptr && at < count ? (int)(at < 0 ? 0 : at) : 0x7fffffff;
  }
  // How many of the split's keys query vector v attends.
  BB_DEV int limit(const Int4DecodeParams& p, int v) const {
    if (!p.causal) return count;
    const int64_t seen = attended(p, n, token_of(p, v)) - begin;
    return (int)(seen < 0 ? 0 : seen < count ? seen : count);
  }
};

// The rest of a split's last chunks, once they have landed: the params that no load brought or that no key has, and the new
// rows.
template <int D, bool F16, int CH>
BB_DEV void complete(const Int4DecodeParams& p, const Part& part, const Stream<D>& in, int c, int g, int lane, uint8_t* s) {
  if ((c + 1) * CH <= part.count && (c + 1) * CH <= part.new_first) return;
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): V too
  wave_fence();
  if ((c + 1) * CH > part.count) {
    if constexpr (D == 64) {
      // an odd last key's params share their 16-byte piece with a row past the range: read them apart
      if ((part.count & 1) && lane < 4) {
        const uint32_t* src = (lane & 2 ? in.vp : in.kp) + 2 * (part.count - 1) + (lane & 1);
        *reinterpret_cast<uint32_t*>(s + (lane & 2 ? kVp : kKp) + param_at<D>(part.count - 1 - c * CH) + 4 * (lane & 1)) = *src;
      }
    }
    // scale and minimum 0 for the V rows past the end, whatever lies there (a probability of 0 times NaN is NaN)
#pragma unroll
    for (int key = lane; key < CH; key += 64)
      if (c * CH + key >= part.count) {
#pragma unroll
        for (int t = 0; t < D / kGroup; ++t) *reinterpret_cast<uint32_t*>(s + kVp + param_at<D>(key) + 4 * t) = 0u;
      }
  }
  if ((c + 1) * CH > part.new_first)
    append_rows<D, F16, CH>(p, part.raw, part.begin, c * CH, part.count, g, lane, s);
  wave_fence();
}

// What a wave leaves in its own LDS when its chunks are done: NV vectors' maxima, sums, minima's parts per column group, and
// the rest of their outputs (rows of D + 4 floats, so that the vectors lie on other banks).
template <int D, int NV>
struct WaveState {
  float m[NV], l[NV], z[NV][D / kGroup], o[NV][D + 4];
};

// The four waves' states under one maximum: the split's partial, or with one split the output.
template <int D, bool F16, int NV>
BB_DEV void finish(const Int4DecodeParams& p, const Part& part, const uint8_t (*sm)[2][kStage], int R, int v0, int g,
                   int split, int tid) {
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < R * (D / 4); i += kThreads) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4)), v = v0 + r, t = token_of(p, v), hd = g * p.G + v - t * p.G;
    float M = kLowest, L = 0.0f;
    f32x4_t O = {0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, reinterpret_cast<const WaveState<D, NV>*>(sm[w])->m[r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const WaveState<D, NV>* f = reinterpret_cast<const WaveState<D, NV>*>(sm[w]);
      const float wt = fast_exp2(f->m[r] - M), z = f->z[r][d / kGroup];
      const f32x4_t o = *reinterpret_cast<const f32x4_t*>(&f->o[r][d]);
      L += wt * f->l[r];
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(wt, o[e] + z, O[e]);
    }
    if (p.n_splits == 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = attended(p, part.n, t) > 0 ? O[e] / L : 0.0f;
      *reinterpret_cast<u32x2_t*>(p.out + t * p.so0 + hd * p.so1 + d) = u32x2_t{pack2<F16>(O[0], O[1]), pack2<F16>(O[2], O[3])};
    } else {
      float* dst = p.part + (((int64_t)t * p.H + hd) * p.n_splits + split) * int4_part_row(D);
      *reinterpret_cast<f32x4_t*>(dst + d) = O;
      if (d == 0) { dst[D] = M; dst[D + 1] = L; }
    }
  }
}

// A query's 8 columns w as an operand fragment in the codes' order: element 2 m / 2 m + 1 = column m / m + 4.
BB_DEV bf16x8_t query_fragment(u32x4_t w, bool on) {
  w = on ? w : u32x4_t{0, 0, 0, 0};
  return as_bf16x8(u32x4_t{(w[0] & 0xffffu) | (w[2] << 16), (w[0] >> 16) | (w[2] & 0xffff0000u),
                           (w[1] & 0xffffu) | (w[3] << 16), (w[1] >> 16) | (w[3] & 0xffff0000u)});
}
template <bool F16>
BB_DEV bf16x8_t fragment_of_ones() {
  constexpr uint32_t one = F16 ? 0x3c003c00u : 0x3f803f80u;
  return as_bf16x8(u32x4_t{one, one, one, one});
}

// Probabilities times scales as operands of 16 bits: two bf16 terms each (off by 2^-17 at most). bf16 whatever the model's type
// (an fp16 product could fall below its range); one term alone would double the error of a bf16 output (2.7e-3 of its norm
// instead of 1.6e-3, measured) and is coarser than an fp16 one. With two the sums are off by 5e-6 of the output's norm, a
// fortieth of an fp16 output's own rounding; a third would bring that to 1e-6 (8111 rows) and costs 3 to 7 % of the kernel.
// The rests are dot products of the first terms with (-1, 0) and (0, -1) added to the numbers, one instruction each. (The asm
// keeps the compiler from rounding a number a second time to have its first term alone, and (-1, 0) in a register: as an inline
// constant the instruction reads it as (0, -1).)
BB_DEV u32x2_t two_terms(float q0, float q1) {
  uint32_t hi = pack_bf16x2(q0, q1), first = 0x0000bf80u;
  asm("" : "+v"(hi));
  asm("" : "+s"(first));
  return u32x2_t{hi, pack_bf16x2(dot2<false>(hi, first, q0), dot2<false>(hi, 0xbf800000u, q1))};
}

// Up to 4 query vectors.
//   scores  Lane (k, a) of 16 x 4 holds the 16 bytes of group a of key k (head_dim 64: group a & 1 of the key in half
//           a >> 1). The query operand is block-diagonal: row 4 a + h holds group a of query h where the lane's quarter is
//           a and zero elsewhere, so the four 16x16x32 products of a 1 KB piece leave in lane (k, a) the four queries' sums
//           over its own group. One (s, z) word per lane turns them into scores; three lane swaps sum the groups and
//           leave lane (k, a) with the whole score of query a alone, so that no lane's exponential is idle.
//   values  The probabilities times the scales of column group t go to column 4 t + h of the operand, so one product serves
//           all groups (the columns of a product whose rows are another group are not used).
// What bounds it, measured: 131072 rows x 8 KV heads x 4 heads of 128 (168 MB) take 34.2 us a call with the merge, 4.9 TB/s, in
// a queue of calls (traced one by one, which adds each kernel's start and end, 31.0 and 4.0); with the arithmetic taken out the
// loads alone and the merge take 30.3 together. The rest is the first chunks' way from memory (a wave's first chunk is there
// after 3.8 us) and the last chunks' arithmetic, which nothing overlaps: with two stages a wave 160 KB a CU are in flight from
// the start, and a split is 8 chunks a wave here. 64 splits a head, two workgroups per CU: 35.3 us with the merge where 32 splits
// took 34.0 to 36.0, 48 splits 38.5, 96 splits 38.6; plain instead of non-temporal loads 39.1 against 37.3 when that was tried.
// The same 10 us past a streaming read's time weigh more where there is less to read: head_dim 64, 100000 rows x 8 heads (64 MB)
// 20.4 us, 11 past it, a split's 12.25 chunks being four rounds for one of its waves and three for the others.
template <int D, bool F16>
__global__ __launch_bounds__(kThreads, 2) void int4_decode_kernel(Int4DecodeParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[kWaves][2][kStage];
  constexpr int CH = D == 128 ? 64 : 128;      // keys of a chunk
  constexpr int W = D == 128 ? 1 : 2;          // queries whose scores a lane ends up with
  constexpr int NG = D / kGroup, NDB = D / 16; // column groups, blocks of 16 columns
  constexpr int HV = CH / 64;                  // 64-key halves of a chunk
  constexpr int PROW = 2 * CH + 16;            // bytes of a probability row in LDS (16 more: rows on other banks)
  const int split = blockIdx.x, g = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), k = lane & 15, a = lane >> 4, R = p.T * p.G;
  const Part part(p, split);
  if (part.count == 0 && p.n_splits > 1) return;  // no partial: the merge knows the live splits

  const Stream<D> in(p, g, part.begin, part.count, lane);
  in.fetch_k(sm[wave][0], wave);
  in.fetch_v(sm[wave][0], wave);
  u32x4_t qw[4];
  const bool on = (k >> 2) == a && (k & 3) < R;
  {
    const int v = (k & 3) < R ? k & 3 : 0, t = token_of(p, v);
    const uint16_t* qr = p.q + t * p.sq0 + (g * p.G + v - t * p.G) * p.sq1 + kGroup * (D == 128 ? a : a & 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) qw[j] = ld16(qr + 8 * j);
  }
  in.fetch_k(sm[wave][1], wave + kWaves);
  in.fetch_v(sm[wave][1], wave + kWaves);
  const int chunks = (part.count + CH - 1) / CH;

  bf16x8_t qa[4];  // fragment i: columns 8 i .. 8 i + 7 of the lane's group
  f32x4_t qs = {0, 0, 0, 0}, qb = {0, 0, 0, 0};  // sums of the queries' groups times p.c, and what the bases add to the products
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    qa[i] = query_fragment(qw[i], on);
    qs = mma16<F16>(qa[i], fragment_of_ones<F16>(), qs);
    qb = mma16<F16>(qa[i], Codes<F16>::bases(), qb);
  }
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    qs[h] *= p.c;
    qb[h] = -qb[h];
  }
  uint32_t kread[2], kpread, vpread;  // where the reads of a stage start
  if constexpr (D == 128) {
    kread[0] = kread[1] = 1024 * (k >> 2) + 64 * (k & 3) + 16 * (a ^ (-(k >> 2) & 3));
    kread[1] += 256;
    kpread = kKp + 16 * k + 4 * a;
    vpread = kVp + 16 * k;
  } else {
    const uint32_t r = 2048 * (a >> 1) + 512 * (k >> 2) + 32 * (k & 3) + 16 * (a & 1);
    kread[0] = r + 128 * (k >> 3);
    kread[1] = r + 128 * ((k >> 3) ^ 1);
    kpread = kKp + 256 * (a >> 1) + 16 * k + 4 * (a & 1);
    vpread = kVp + 256 * (a >> 1) + 16 * k;
  }
  const int key_k = (D == 128 ? 0 : 64 * (a >> 1)) + key_of_lane(k);
  int lim[W];
#pragma unroll
  for (int w = 0; w < W; ++w) lim[w] = part.limit(p, D == 128 ? a : (a & 1) + 2 * w);
  const int fewest = part.limit(p, 0);  // the first token's is the smallest
  const float up01 = prob_up(k % 2 == 0);  // a lane's steps 0 and 1: the first pair of its operand's eight keys where k is even

  float m[W], l[W], zs[W][NG];
  f32x4_t o[NDB];
#pragma unroll
  for (int w = 0; w < W; ++w) {
    m[w] = kLowest;
    l[w] = 0.0f;
#pragma unroll
    for (int t = 0; t < NG; ++t) zs[w][t] = 0.0f;
  }
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = f32x4_t{0, 0, 0, 0};

  const Codes<F16> k_codes;
  const ValueCodes v_codes;
  int st = 0;
  for (int c = wave; c < chunks; c += kWaves, st ^= 1) {
    __builtin_amdgcn_s_waitcnt(0x0F7F);  // vmcnt(15): this chunk's K has landed; its V and the next chunk may be in flight
    wave_fence();
    uint8_t* s = sm[wave][st];
    complete<D, F16, CH>(p, part, in, c, g, lane, s);

    float x[W][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const u32x4_t kw = *reinterpret_cast<const u32x4_t*>(s + kread[u >> 1] + (D == 128 ? 512 : 256) * (u & 1));
      const uint32_t kp = *reinterpret_cast<const uint32_t*>(s + kpread + (D == 128 ? 256 * u : 512 * (u & 1) + 8 * (u >> 1)));
      const float sc = mul_lo(p.c, kp);
      f32x4_t acc = qb;
#pragma unroll
      for (int i = 0; i < 4; ++i) acc = mma16<F16>(qa[i], k_codes(kw[i]), acc);
      float y[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) y[h] = fmaf(sc, acc[h], mul_hi(qs[h], kp));
      if constexpr (D == 128) {
        x[0][u] = sum_rows16(sum_rows32(y[0], y[2]), sum_rows32(y[1], y[3]));
      } else {
        x[0][u] = sum_rows16(y[0], y[1]);
        x[W - 1][u] = sum_rows16(y[2], y[3]);
      }
    }
    if (c * CH + CH > fewest) {
      asm volatile("; a branch: most chunks are whole");
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (c * CH + key_k + key_of_step(u) >= lim[w]) x[w][u] = -__builtin_huge_valf();
    }
    float pr[W][4];
    float most = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        pr[w][u] = fast_exp2(x[w][u] - m[w]);
        most = fmaxf(most, pr[w][u]);
      }
    if (__builtin_amdgcn_ballot_w64(most > kOver)) {
      float alpha[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        float mx = row_max(fmaxf(fmaxf(x[w][0], x[w][1]), fmaxf(x[w][2], x[w][3])));
        if constexpr (D == 64) mx = xhalf_max(mx);
        const float mn = fmaxf(m[w], mx);
        alpha[w] = fast_exp2(m[w] - mn);
        m[w] = mn;
        l[w] *= alpha[w];
#pragma unroll
        for (int u = 0; u < 4; ++u) pr[w][u] = fast_exp2(x[w][u] - mn);
#pragma unroll
        for (int t = 0; t < NG; ++t) zs[w][t] *= alpha[w];
      }
      // column 4 t + h of the sums belongs to query h
      float al[4];
#pragma unroll
      for (int h = 0; h < 4; ++h)
        al[h] = D == 128 ? lane_value(alpha[0], 16 * h) : lane_value(alpha[W - 1 ? h >> 1 : 0], 16 * (h & 1));
      const float ac = k & 2 ? (k & 1 ? al[3] : al[2]) : (k & 1 ? al[1] : al[0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db][e] *= ac;
      }
    }
    __builtin_amdgcn_s_waitcnt(0x0F7A);  // vmcnt(10): this chunk's V too
    wave_fence();
    uint32_t vp[4][NG];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if constexpr (D == 128) {
        const u32x4_t r = *reinterpret_cast<const u32x4_t*>(s + vpread + 256 * u);
#pragma unroll
        for (int t = 0; t < NG; ++t) vp[u][t] = r[t];
      } else {
        const u32x2_t r = *reinterpret_cast<const u32x2_t*>(s + vpread + 512 * (u & 1) + 8 * (u >> 1));
        vp[u][0] = r[0];
        vp[u][1] = r[1];
      }
    }
    // probabilities times V scales, [4 t + h][key], in the space of the K rows
    wave_fence();
#pragma unroll
    for (int w = 0; w < W; ++w) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        l[w] += pr[w][u];
#pragma unroll
        for (int t = 0; t < NG; ++t) zs[w][t] = fmaf(pr[w][u], f16_hi(vp[u][t]), zs[w][t]);
        pr[w][u] *= u < 2 ? up01 : prob_up(false);
      }
#pragma unroll
      for (int t = 0; t < NG; ++t) {
        float q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = mul_lo(pr[w][u], vp[u][t]);
        const int col = D == 128 ? 4 * t + a : 4 * t + (a & 1) + 2 * w;
        const u32x2_t q01 = two_terms(q[0], q[1]), q23 = two_terms(q[2], q[3]);
        uint8_t* dst = s + col * PROW + (D == 128 ? 0 : 128 * (a >> 1)) + 8 * k;
        *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{q01[0], q23[0]};
        *reinterpret_cast<u32x2_t*>(dst + 4 * NG * PROW) = u32x2_t{q01[1], q23[1]};
      }
    }
    wave_fence();
    bf16x8_t pb[2 * HV], pl[2 * HV];
    {
      const uint8_t* src = s + (D == 128 ? k : k & 7) * PROW + 32 * a;  // head_dim 64: columns 8..15 repeat and are not used
#pragma unroll
      for (int j = 0; j < 2 * HV; ++j) {
        pb[j] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(src + 128 * (j >> 1) + 16 * (j & 1)));
        pl[j] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(src + 4 * NG * PROW + 128 * (j >> 1) + 16 * (j & 1)));
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the probabilities are read, the K rows' space is free
    wave_fence();
    in.fetch_k(s, c + 2 * kWaves);
#pragma unroll
    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        const v2i_t t = read_tr4(s + kVq + v_block_at<D>(k, a, hv, db));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bf16x8_t vf = v_codes((uint32_t)(j ? t.y : t.x));
          o[db] = mma16_bf16(vf, pb[2 * hv + j], o[db]);
          o[db] = mma16_bf16(vf, pl[2 * hv + j], o[db]);
        }
      }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the V rows are read
    wave_fence();
    in.fetch_v(s, c + 2 * kWaves);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): nothing lands in LDS any more

  WaveState<D, 4>* mine = reinterpret_cast<WaveState<D, 4>*>(sm[wave]);
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int v = D == 128 ? a : (a & 1) + 2 * w;
    float sum = row_sum(l[w]);
    if constexpr (D == 64) sum = xhalf_sum(sum);
#pragma unroll
    for (int t = 0; t < NG; ++t) {
      float z = row_sum(zs[w][t]);
      if constexpr (D == 64) z = xhalf_sum(z);
      if (k == 0) mine->z[v][t] = z;
    }
    if (k == 0) {
      mine->m[v] = m[w];
      mine->l[v] = sum;
    }
  }
  // lane (4 t + h, a) holds columns 16 db + 4 a .. + 3 of query h, those of group t valid: blocks 2 t and 2 t + 1
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    f32x4_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float lo = k & 4 ? o[2 + j][e] : o[j][e];
      if constexpr (D == 128) lo = k & 8 ? (k & 4 ? o[6 + j][e] : o[4 + j][e]) : lo;
      r[e] = lo * kSumDown;
    }
    if (D == 128 || k < 8) *reinterpret_cast<f32x4_t*>(&mine->o[k & 3][32 * (k >> 2) + 16 * j + 4 * a]) = r;
  }
  finish<D, F16, 4>(p, part, sm, R, 0, g, split, tid);
}

// 5 and more query vectors, 16 of them a pass: column k of every product is vector k.
//   scores  Rows are keys: lane (k, a) reads word a of every group of key k as the codes' operand, one product per group, and is
//           left with vector k's sums over keys 4 a .. 4 a + 3 of the step, to which it applies those keys' (s, z).
//   values  The lane's probabilities are the operand of the values' products as they are: with keys in the order of key_of_lane
//           and key_of_step, a lane's 16 keys of 64 are those whose V codes the transposing read hands to its quarter. So no
//           probability passes through LDS, and the maxima, sums and minima's parts stay with one vector per lane.
// The VALU bounds it: about 680 instructions a chunk (codes to operands 225, probabilities times scales into two terms 190), 3000
// cycles on a SIMD. 16 vectors x 8 KV heads x 128 over 32768 rows (42 MB) take 16.6 us traced; a wave's median, in us at 2.4 GHz:
// 2.5 until its first 20 loads are issued (the other waves of the CU issue theirs as well), 4.0 until the first chunk is
// there, 3.9 for that chunk (the loop's code comes in with it, and the SIMD's other wave works on its own), 2.6 for the second,
// 1.4 for the states and the partials; the slowest wave ends 1 later, and the launch is the rest. Over 131072 rows 42.3 us with
// the merge (4.0 TB/s). Each pass of 16 vectors reads and unpacks the cache again: 64 vectors over 131072 rows 154 us. With 4
// vectors this kernel is slower than the one above (131072 rows 40.2 us against 36.1 with the merge, 512 rows 8.1 against 6.9;
// head_dim 64, 100000 rows 24.7 against 20.2).
template <int D, bool F16>
__global__ __launch_bounds__(kThreads, 2) void int4_decode_wide_kernel(Int4DecodeParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[kWaves][2][kStage];
  constexpr int CH = D == 128 ? 64 : 128;
  constexpr int NG = D / kGroup, NDB = D / 16, HV = CH / 64;
  const int split = blockIdx.x, g = blockIdx.y, v0 = blockIdx.z * kVecs, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), k = lane & 15, a = lane >> 4;
  const int R = p.T * p.G - v0 < kVecs ? p.T * p.G - v0 : kVecs;
  const Part part(p, split);
  if (part.count == 0 && p.n_splits > 1) return;

  const Stream<D> in(p, g, part.begin, part.count, lane);
  in.fetch_k(sm[wave][0], wave);
  in.fetch_v(sm[wave][0], wave);
  u32x4_t qw[NG];  // vector k, columns 8 a .. 8 a + 7 of every group
  {
    const int v = v0 + (k < R ? k : 0), t = token_of(p, v);
    const uint16_t* qr = p.q + t * p.sq0 + (g * p.G + v - t * p.G) * p.sq1 + 8 * a;
#pragma unroll
    for (int j = 0; j < NG; ++j) qw[j] = ld16(qr + kGroup * j);
  }
  in.fetch_k(sm[wave][1], wave + kWaves);
  in.fetch_v(sm[wave][1], wave + kWaves);
  const int chunks = (part.count + CH - 1) / CH;

  // qz: the group sums as three bf16 terms each (24 bits), so that one product per step adds up z times them over the groups,
  // z in two terms (its 11 bits); lane (k, a) holds vector k's group a (head_dim 64: a < 2)
  bf16x8_t qa[NG], qz;
  f32x4_t qb[NG];  // what the bases add to the sums, negative
  {
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      qa[j] = query_fragment(qw[j], k < R);
      const f32x4_t c = mma16<F16>(fragment_of_ones<F16>(), qa[j], f32x4_t{0, 0, 0, 0});  // every row: vector k's sum
      sum = a == j ? c[0] : sum;
      qb[j] = mma16<F16>(Codes<F16>::bases(), qa[j], f32x4_t{0, 0, 0, 0});
#pragma unroll
      for (int e = 0; e < 4; ++e) qb[j][e] = -qb[j][e];
    }
    u32x4_t w = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const uint32_t top = __float_as_uint(sum) & 0xffff0000u;
      w[j] = top | (top >> 16);
      sum -= __uint_as_float(top);
    }
    qz = as_bf16x8(w);
  }
  uint32_t kread[4];  // head_dim 128: by group; 64: by u >> 1
#pragma unroll
  for (int j = 0; j < 4; ++j)
    kread[j] = D == 128 ? 1024 * (k >> 2) + 64 * (k & 3) + 16 * (j ^ (-(k >> 2) & 3)) + 4 * a
                        : 512 * (k >> 2) + 32 * (k & 3) + 128 * ((k >> 3) ^ (j & 1)) + 4 * a;
  const int lim = part.limit(p, v0 + k), fewest = part.limit(p, v0);

  float m = kLowest, l = 0.0f, zs[NG];
  f32x4_t o[NDB];
#pragma unroll
  for (int db = 0; db < NDB; ++db) o[db] = f32x4_t{0, 0, 0, 0};
#pragma unroll
  for (int t = 0; t < NG; ++t) zs[t] = 0.0f;

  const Codes<F16> k_codes;
  const ValueCodes v_codes;
  // the NG params words of key 16 a + 8 (e >> 1) + 2 (e & 1) + key_of_step(u) of half hv, from the stage's K or V params
  auto params = [&](const uint8_t* at, int hv, int u, int e, uint32_t (&w)[NG]) {
    if constexpr (D == 128) {
      const u32x4_t r = *reinterpret_cast<const u32x4_t*>(at + 256 * u + 64 * a + 16 * e);
#pragma unroll
      for (int t = 0; t < NG; ++t) w[t] = r[t];
    } else {
      const u32x2_t r = *reinterpret_cast<const u32x2_t*>(at + 512 * (u & 1) + 256 * hv + 64 * a + 16 * e + 8 * (u >> 1));
      w[0] = r[0];
      w[1] = r[1];
    }
  };
  int st = 0;
  for (int c = wave; c < chunks; c += kWaves, st ^= 1) {
    __builtin_amdgcn_s_waitcnt(0x0F7F);  // vmcnt(15): this chunk's K has landed; its V and the next chunk may be in flight
    wave_fence();
    uint8_t* s = sm[wave][st];
    complete<D, F16, CH>(p, part, in, c, g, lane, s);

    float x[HV][4][4];  // [half][step][key of the lane's four]
#pragma unroll
    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float z = f16_hi(*reinterpret_cast<const uint32_t*>(
            s + kKp + 16 * k + (D == 128 ? 256 * u + 4 * a : 512 * (u & 1) + 256 * hv + 8 * (u >> 1) + 4 * (a & 1))));
        const uint32_t top = __float_as_uint(z) & 0xffff0000u;
        const uint32_t zw = (top >> 16) | (__float_as_uint(z - __uint_as_float(top)) & 0xffff0000u);
        const f32x4_t y = mma16_bf16(as_bf16x8(u32x4_t{zw, zw, zw, 0u}), qz, f32x4_t{0, 0, 0, 0});
#pragma unroll
        for (int e = 0; e < 4; ++e) x[hv][u][e] = y[e];
        f32x4_t acc[NG];
#pragma unroll
        for (int t = 0; t < NG; ++t) {
          const uint32_t kw = *reinterpret_cast<const uint32_t*>(
              s + (D == 128 ? kread[t] + 512 * (u & 1) + 256 * (u >> 1) : kread[u >> 1] + 2048 * hv + 256 * (u & 1) + 16 * t));
          acc[t] = mma16<F16>(k_codes(kw), qa[t], qb[t]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          uint32_t kp[NG];
          params(s + kKp, hv, u, e, kp);
#pragma unroll
          for (int t = 0; t < NG; ++t) x[hv][u][e] = fmaf(f16_lo(kp[t]), acc[t][e], x[hv][u][e]);
          x[hv][u][e] *= p.c;  // rounded: as one fma with the maximum, keys that tie at a score past 2^30 would differ
        }
      }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the K rows are read, their space is free
    wave_fence();
    in.fetch_k(s, c + 2 * kWaves);
    if (c * CH + CH > fewest) {
      asm volatile("; a branch: most chunks are whole");
#pragma unroll
      for (int hv = 0; hv < HV; ++hv)
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (c * CH + 64 * hv + 16 * a + 8 * (e >> 1) + 2 * (e & 1) + key_of_step(u) >= lim)
              x[hv][u][e] = -__builtin_huge_valf();
    }
    float pr[HV][4][4];
    float most = 0.0f;
#pragma unroll
    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          pr[hv][u][e] = fast_exp2(x[hv][u][e] - m);
          most = fmaxf(most, pr[hv][u][e]);
        }
    if (__builtin_amdgcn_ballot_w64(most > kOver)) {
      float mx = x[0][0][0];
#pragma unroll
      for (int i = 1; i < 16 * HV; ++i) mx = fmaxf(mx, x[i >> 4][(i >> 2) & 3][i & 3]);
      const float mn = fmaxf(m, quarters_max(mx)), alpha = fast_exp2(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 16 * HV; ++i)
        pr[i >> 4][(i >> 2) & 3][i & 3] = fast_exp2(x[i >> 4][(i >> 2) & 3][i & 3] - mn);
#pragma unroll
      for (int t = 0; t < NG; ++t) zs[t] *= alpha;
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[db][e] *= alpha;
    }
#pragma unroll
    for (int i = 0; i < 16 * HV; ++i) l += pr[i >> 4][(i >> 2) & 3][i & 3];

    __builtin_amdgcn_s_waitcnt(0x0F7F);  // vmcnt(15): this chunk's V; the next chunk and the K behind it may be in flight
    wave_fence();
#pragma unroll
    for (int hv = 0; hv < HV; ++hv) {
      v2i_t vw[NDB];
#pragma unroll
      for (int db = 0; db < NDB; ++db) vw[db] = read_tr4(s + kVq + v_block_at<D>(k, a, hv, db));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // element 2 (2 (e & 1) + (u >> 1)) + (u & 1) of operand j is key (u, e) with e >> 1 = j
        uint32_t vp[4][2][NG];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int e = 0; e < 2; ++e) params(s + kVp, hv, u, 2 * j + e, vp[u][e]);
#pragma unroll
        for (int t = 0; t < NG; ++t) {
          u32x4_t hi, lo;
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const float p0 = pr[hv][2 * i][2 * j + e], p1 = pr[hv][2 * i + 1][2 * j + e];
              const uint32_t w0 = vp[2 * i][e][t], w1 = vp[2 * i + 1][e][t];
              const float up = prob_up(e == 0 && i == 0);
              const u32x2_t q = two_terms(mul_lo(p0 * up, w0), mul_lo(p1 * up, w1));
              hi[2 * e + i] = q[0];
              lo[2 * e + i] = q[1];
              zs[t] = fmaf(p0, f16_hi(w0), fmaf(p1, f16_hi(w1), zs[t]));
            }
#pragma unroll
          for (int db = 2 * t; db < 2 * t + 2; ++db) {
            const bf16x8_t vf = v_codes((uint32_t)(j ? vw[db].y : vw[db].x));
            o[db] = mma16_bf16(vf, as_bf16x8(hi), o[db]);
            o[db] = mma16_bf16(vf, as_bf16x8(lo), o[db]);
          }
        }
      }
    }
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the V rows are read
    wave_fence();
    in.fetch_v(s, c + 2 * kWaves);
  }
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): nothing lands in LDS any more

  WaveState<D, kVecs>* mine = reinterpret_cast<WaveState<D, kVecs>*>(sm[wave]);
  l = quarters_sum(l);
#pragma unroll
  for (int t = 0; t < NG; ++t) {
    zs[t] = quarters_sum(zs[t]);
    if (a == 0) mine->z[k][t] = zs[t];
  }
  if (a == 0) {
    mine->m[k] = m;
    mine->l[k] = l;
  }
#pragma unroll
  for (int db = 0; db < NDB; ++db) {
    f32x4_t r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = o[db][e] * kSumDown;
    *reinterpret_cast<f32x4_t*>(&mine->o[k][16 * db + 4 * a]) = r;
  }
  finish<D, F16, kVecs>(p, part, sm, R, v0, g, split, tid);
}

// The partials of the live splits under one maximum: a workgroup per (query vector, 32 columns), thread (4 columns, group)
// folding every 16th split, 4 loaded at a time; the groups then combine through LDS. Latency bounds it (2.2 to 4 us for
// 0.5 to 4 MB). GPU time of decode and merge over 8111 rows, 32 splits: 11.4 us with 8 groups, 11.6 with 16, 12.1 with 32, 12.6
// with 64; over 131072 rows, 64 splits, 8 and 16 are even and 64 takes 1 us more.
constexpr int kMergeCols = 32, kMergeLanes = kMergeCols / 4, kMergeGroups = 16, kMergePer = 4;
template <int D, bool F16>
__global__ __launch_bounds__(kMergeLanes * kMergeGroups) void int4_merge_kernel(Int4DecodeParams p) {
  __shared__ __attribute__((aligned(16))) float sm_o[kMergeGroups][kMergeCols];
  __shared__ float sm_m[kMergeGroups], sm_l[kMergeGroups];
  const int v = blockIdx.x, c = 4 * (threadIdx.x % kMergeLanes), grp = threadIdx.x / kMergeLanes, d0 = kMergeCols * blockIdx.y;
  int64_t n = p.n, len = p.len;
  if (p.n_dev) {
    n = live_length(p, *p.n_dev);
    len = split_keys(p, n);
  }
  const int live = (int)((n + len - 1) / len);
  const float* base = p.part + (int64_t)v * p.n_splits * int4_part_row(D);
  float M = kLowest, L = 0.0f;
  f32x4_t O = {0, 0, 0, 0};
  for (int i0 = grp; i0 < live; i0 += kMergeGroups * kMergePer) {
    float mv[kMergePer], lv[kMergePer];
    f32x4_t ov[kMergePer];
#pragma unroll
    for (int i = 0; i < kMergePer; ++i) {
      const int s = i0 + kMergeGroups * i;
      const bool ok = s < live;
      const float* r = base + (int64_t)(ok ? s : i0) * int4_part_row(D);
      mv[i] = ok ? r[D] : kLowest;
      lv[i] = ok ? r[D + 1] : 0.0f;
      ov[i] = *reinterpret_cast<const f32x4_t*>(r + d0 + c);
    }
    float mn = M;
#pragma unroll
    for (int i = 0; i < kMergePer; ++i) mn = fmaxf(mn, mv[i]);
    const float al = fast_exp2(M - mn);
    L *= al;
#pragma unroll
    for (int e = 0; e < 4; ++e) O[e] *= al;
#pragma unroll
    for (int i = 0; i < kMergePer; ++i) {
      const float w = i0 + kMergeGroups * i < live ? fast_exp2(mv[i] - mn) : 0.0f;
      L += w * lv[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(w, ov[i][e], O[e]);
    }
    M = mn;
  }
  *reinterpret_cast<f32x4_t*>(&sm_o[grp][c]) = O;
  if (c == 0) { sm_m[grp] = M; sm_l[grp] = L; }
  __syncthreads();
  if (threadIdx.x < kMergeCols) {
    const int d = threadIdx.x;
    float mx = sm_m[0];
#pragma unroll
    for (int i = 1; i < kMergeGroups; ++i) mx = fmaxf(mx, sm_m[i]);
    float lt = 0.0f, ot = 0.0f;
#pragma unroll
    for (int i = 0; i < kMergeGroups; ++i) {
      const float w = fast_exp2(sm_m[i] - mx);
      lt += w * sm_l[i];
      ot += w * sm_o[i][d];
    }
    const int t = v / p.H;
    p.out[t * p.so0 + (v % p.H) * p.so1 + d0 + d] = to16<F16>(attended(p, n, t) > 0 ? ot / lt : 0.0f);
  }
}

template <int D, bool F16>
hipError_t launch_decode_t(const Int4DecodeParams& p, hipStream_t stream) {
  const int vecs = p.T * p.G;
  if (vecs <= 4)
    hipLaunchKernelGGL((int4_decode_kernel<D, F16>), dim3(p.n_splits, p.Hkv), dim3(kThreads), 0, stream, p);
  else
    hipLaunchKernelGGL((int4_decode_wide_kernel<D, F16>), dim3(p.n_splits, p.Hkv, (vecs + kVecs - 1) / kVecs),
                       dim3(kThreads), 0, stream, p);
  if (p.n_splits > 1)
    hipLaunchKernelGGL((int4_merge_kernel<D, F16>), dim3(p.T * p.H, D / kMergeCols),
                       dim3(kMergeLanes * kMergeGroups), 0, stream, p);
  return hipGetLastError();
}

}  // namespace

template <int D>
static hipError_t launch_quantize_d(const Int4Set& s0, const Int4Set& s1, bool two, int kind, int heads, int64_t rows,
                                    hipStream_t stream) {
  const dim3 grid((unsigned)((rows + 4096 / D - 1) / (4096 / D) * heads), two ? 2u : 1u);
  if (kind == kKindF32) hipLaunchKernelGGL((int4_quantize_kernel<D, kKindF32>), grid, dim3(256), 0, stream, s0, s1, heads, rows);
  else if (kind == kKindF16) hipLaunchKernelGGL((int4_quantize_kernel<D, kKindF16>), grid, dim3(256), 0, stream, s0, s1, heads, rows);
  else hipLaunchKernelGGL((int4_quantize_kernel<D, kKindBf16>), grid, dim3(256), 0, stream, s0, s1, heads, rows);
  return hipGetLastError();
}

hipError_t launch_int4_quantize(const Int4Rows& k, const Int4Rows* v, int kind, int heads, int64_t rows, int D,
                                hipStream_t stream) {
  if (rows <= 0 || heads <= 0) return hipSuccess;
  const Int4Set s0{k.x, k.q, k.p, k.sx0, k.sx1, k.sq0, k.sp0};
  const Int4Set s1 = v ? Int4Set{v->x, v->q, v->p, v->sx0, v->sx1, v->sq0, v->sp0} : s0;
  switch (D) {
    case 32: return launch_quantize_d<32>(s0, s1, v != nullptr, kind, heads, rows, stream);
    case 64: return launch_quantize_d<64>(s0, s1, v != nullptr, kind, heads, rows, stream);
    case 128: return launch_quantize_d<128>(s0, s1, v != nullptr, kind, heads, rows, stream);
    case 256: return launch_quantize_d<256>(s0, s1, v != nullptr, kind, heads, rows, stream);
    default: return hipErrorInvalidValue;
  }
}

template <int D>
static hipError_t launch_dequantize_d(const Int4ReadSet& s0, const Int4ReadSet& s1, bool two, int kind, int heads,
                                      int64_t rows, hipStream_t stream) {
  const dim3 grid((unsigned)((rows + 2048 / D - 1) / (2048 / D)), (unsigned)heads, two ? 2u : 1u);
  hipLaunchKernelGGL(int4_dequantize_kernel<D>, grid, dim3(256), 0, stream, s0, s1, kind, rows);
  return hipGetLastError();
}

hipError_t launch_int4_dequantize(const Int4Rows& k, const Int4Rows* v, int kind, int heads, int64_t rows, int D,
                                  hipStream_t stream) {
  if (rows <= 0 || heads <= 0) return hipSuccess;
  const Int4ReadSet s0{k.q, k.p, const_cast<void*>(k.x), k.sq0, k.sp0};
  const Int4ReadSet s1 = v ? Int4ReadSet{v->q, v->p, const_cast<void*>(v->x), v->sq0, v->sp0} : s0;
  switch (D) {
    case 32: return launch_dequantize_d<32>(s0, s1, v != nullptr, kind, heads, rows, stream);
    case 64: return launch_dequantize_d<64>(s0, s1, v != nullptr, kind, heads, rows, stream);
    case 128: return launch_dequantize_d<128>(s0, s1, v != nullptr, kind, heads, rows, stream);
    case 256: return launch_dequantize_d<256>(s0, s1, v != nullptr, kind, heads, rows, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_int4_decode(const Int4DecodeParams& p, hipStream_t stream) {
  if (p.D == 64) return p.f16 ? launch_decode_t<64, true>(p, stream) : launch_decode_t<64, false>(p, stream);
  return p.f16 ? launch_decode_t<128, true>(p, stream) : launch_decode_t<128, false>(p, stream);
}

}  // namespace bb
