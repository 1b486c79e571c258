// KV cache in 4 bits: the write, the read back, and the exact attention of a few query tokens over the packed rows.
//
// A row of D elements is D / 32 groups of 32. Per group, on values clamped to +-65504 (NaN counts as 0):
//   z = fp16(min), s = fp16(max((max - z) / 15, 0)), code = rint((x - z) / s) clamped to 0..15 (0 where s = 0),
// each operation in fp32; the value is s * code + z in fp32 (s * code is exact). s and z are rounded before the codes are
// taken, so the codes make up for their rounding. Byte b of a packed row holds elements 2 b (low four bits) and 2 b + 1.
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
BB_DEV uint32_t f16_bits(float f) { return __builtin_bit_cast(uint16_t, (_Float16)f); }  // round to nearest even

// Eight elements of a row at x (16-byte aligned), in fp32.
BB_DEV void load8(const void* x, int64_t off, int kind, float (&v)[8]) {
  if (kind == kKindF32) {
    const float* p = reinterpret_cast<const float*>(x) + off;
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p), b = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
  } else {
    const u32x4_t a = ld16(reinterpret_cast<const uint16_t*>(x) + off);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = kind == kKindF16 ? f16_lo(a[i]) : bf16_to_f32((uint16_t)(a[i] & 0xffffu));
      v[2 * i + 1] = kind == kKindF16 ? f16_hi(a[i]) : bf16_to_f32((uint16_t)(a[i] >> 16));
    }
  }
}

// Quantises the 8 elements v of a lane; the 4 lanes of an aligned quad hold one group and all take part. Returns the 8
// codes, little-endian, and the group's (s, z) as packed fp16.
BB_DEV uint32_t quant8_4bit(float (&v)[8], uint32_t& param) {
  float lo = kF16Max, hi = -kF16Max;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = v[i] == v[i] ? fminf(fmaxf(v[i], -kF16Max), kF16Max) : 0.0f;
    lo = fminf(lo, v[i]);
    hi = fmaxf(hi, v[i]);
  }
  lo = fminf(lo, dpp_mov<0xB1>(lo));
  hi = fmaxf(hi, dpp_mov<0xB1>(hi));
  lo = fminf(lo, dpp_mov<0x4E>(lo));
  hi = fmaxf(hi, dpp_mov<0x4E>(hi));
  const uint32_t zb = f16_bits(lo);
  const float z = f16_lo(zb);
  const uint32_t sb = f16_bits(fmaxf((hi - z) / 15.0f, 0.0f));
  const float s = f16_lo(sb);
  param = sb | (zb << 16);
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = s > 0.0f ? fminf(fmaxf(rintf((v[i] - z) / s), 0.0f), 15.0f) : 0.0f;
    w |= (uint32_t)c << (4 * i);
  }
  return w;
}

struct Int4Set {  // one tensor's rows and their place in the cache
  const void* x;
  uint8_t* q;
  uint32_t* p;
  int64_t sx0, sx1;  // head and row stride of x (elements)
  int64_t sq0, sp0;  // head strides of q (bytes) and p (groups)
};

// A lane takes 8 elements of a row; blockIdx.y is the head, blockIdx.z the tensor (K, V).
template <int D>
__global__ __launch_bounds__(256) void int4_quantize_kernel(Int4Set s0, Int4Set s1, int kind, int64_t rows) {
  const Int4Set& s = blockIdx.z ? s1 : s0;
  constexpr int LPR = D / 8;
  const int64_t row = (int64_t)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int c = threadIdx.x % LPR, h = blockIdx.y;
  if (row >= rows) return;  // the lanes of a row leave together
  float v[8];
  load8(s.x, h * s.sx0 + row * s.sx1 + 8 * c, kind, v);
  uint32_t param;
  const uint32_t w = quant8_4bit(v, param);
  *reinterpret_cast<uint32_t*>(s.q + h * s.sq0 + row * (D / 2) + 4 * c) = w;
  if (c % 4 == 0) s.p[h * s.sp0 + row * (D / kGroup) + c / 4] = param;
}

struct Int4ReadSet {
  const uint8_t* q;
  const uint32_t* p;
  void* out;  // [heads, rows, D] contiguous
  int64_t sq0, sp0;
};

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
    float* o = reinterpret_cast<float*>(s.out) + off;
    *reinterpret_cast<f32x4_t*>(o) = f32x4_t{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4_t*>(o + 4) = f32x4_t{v[4], v[5], v[6], v[7]};
  } else {
    u32x4_t o;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      o[i] = kind == kKindF16 ? pack2<true>(v[2 * i], v[2 * i + 1]) : pack2<false>(v[2 * i], v[2 * i + 1]);
    st16(reinterpret_cast<uint16_t*>(s.out) + off, o);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Attention over the packed rows, split over the keys. Workgroup (split, KV head, pass): 4 waves against the split's keys,
// wave w taking chunks w, w + 4, ... of 64 keys (128 at head_dim 64); a pass takes up to 16 query vectors (T tokens x G
// heads of the KV head, token-major) in blocks of 4. The length may come from device memory; every launch shape depends on
// host values alone.
//
// Mathematics. With k = s c + z per group of 32 (c the codes), q.k = sum_g s_g (q_g . c_g) + z_g sum(q_g), and
// o = sum_j p_j s_j c_j + sum_j p_j z_j per column group: the codes go to the matrix cores as they are, exact in 16 bits, and
// scales and minima are applied in fp32 to the sums (scores) or to the probabilities (values). A code becomes the 16-bit
// float 16 + c by one shift and one and-or per two codes; the 16s are taken back from the sums.
//
//   scores  Lane (k, a) of 16 x 4 holds the 16 bytes of group a of key k (head_dim 64: group a & 1 of the key in half
//           a >> 1). The query operand is block-diagonal: row 4 a + h holds group a of query h where the lane's quarter is
//           a and zero elsewhere, so the four 16x16x32 products of a 1 KB piece leave in lane (k, a) the four queries' sums
//           over its own group. One (s, z) word per lane turns them into scores; three lane swaps sum the groups and
//           leave lane (k, a) with the whole score of query a alone, so that no lane's exponential is idle.
//   values  V rows are transposed by ds_read_b64_tr_b4 (a lane gets 16 keys of one column). The probabilities times the
//           scales of column group t go to column 4 t + h of the other operand, so one product serves all groups (the
//           columns of a product whose rows are another group are not used). The 16s go with a row of ones.
//
// A chunk's 10 KB (codes and params of K and of V) stream straight into the wave's LDS with ten buffer loads that cover
// whole lines, one chunk ahead. Pieces land so that the operand reads meet no bank twice: see the offsets at each.
constexpr int kVecs = 16;            // query vectors of a pass
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kStage = 10240;        // K codes 4096 | K params 1024 | V codes 4096 | V params 1024
constexpr int kKp = 4096, kVq = 5120, kVp = 9216;
constexpr float kOver = 256.0f;      // a probability past this moves the running maximum

typedef int v2i_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void;

BB_DEV int64_t live_length(const Int4DecodeParams& p) {
  const int64_t n = p.n_dev ? *p.n_dev : p.n;
  return n < 0 ? 0 : n > p.cap ? p.cap : n;
}
// Keys of a split: the live length in equal parts of whole 16 keys (the bytes per CU set the time, so the parts are not
// rounded to chunks).
BB_DEV int64_t split_keys(int64_t n, int n_splits) {
  const int64_t len = ((n + n_splits - 1) / n_splits + 15) & ~(int64_t)15;
  return len < kInt4MinSplit ? kInt4MinSplit : len;
}
// Keys that token t of T attends.
BB_DEV int64_t seen_keys(const Int4DecodeParams& p, int64_t n, int t) { return p.causal ? n - p.T + 1 + t : n; }

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

// Eight codes as 16-bit floats 16 + c, in the order 0, 4, 1, 5, 2, 6, 3, 7 (the halves of the word side by side). 16.0 has
// an ulp of 1/8 in bf16 and 1/64 in fp16, so a code is a shift away from its place in the mantissa.
template <bool F16>
BB_DEV bf16x8_t codes16(uint32_t w) {
  constexpr uint32_t mask = F16 ? 0x03c003c0u : 0x00780078u, base = F16 ? 0x4c004c00u : 0x41804180u;
  constexpr int sh = F16 ? 6 : 3;
  return as_bf16x8(u32x4_t{((w << sh) & mask) | base, ((F16 ? w << 2 : w >> 1) & mask) | base,
                           ((w >> (8 - sh)) & mask) | base, ((w >> (12 - sh)) & mask) | base});
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
BB_DEV float lane_value(float v, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), lane));
}

// LDS written by this wave before is what it reads after (LDS operations of one wave run in order: this orders the compiler).
BB_DEV void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The step's new rows that lie in cache rows [begin, end): quantised there by the threads of a workgroup.
template <int D>
BB_DEV void append_rows(const Int4DecodeParams& p, int64_t n, int64_t begin, int64_t end, int g, int tid) {
  constexpr int LPR = D / 8;
  const int c = tid % LPR;
  for (int i = tid / LPR; i < 2 * p.T; i += kThreads / LPR) {  // the lanes of a row stay together
    const int t = i >> 1, vt = i & 1;
    const int64_t row = n - p.T + t;
    if (row < begin || row >= end) continue;
    float v[8];
    load8(vt ? p.vnew : p.knew, vt ? g * p.svn0 + t * p.svn1 + 8 * c : g * p.skn0 + t * p.skn1 + 8 * c,
          p.f16 ? kKindF16 : kKindBf16, v);
    uint32_t param;
    const uint32_t w = quant8_4bit(v, param);
    uint8_t* q = vt ? p.vq + g * p.svq : p.kq + g * p.skq;
    uint32_t* pp = vt ? p.vp + g * p.svp : p.kp + g * p.skp;
    *reinterpret_cast<uint32_t*>(q + row * (D / 2) + 4 * c) = w;
    if (c % 4 == 0) pp[row * (D / kGroup) + c / 4] = param;
  }
}

// NB: blocks of 4 query vectors. TWO: a probability times a scale goes to the matrix cores as two bf16 terms (16
// significant bits) instead of one.
template <int D, bool F16, int NB, bool TWO>
__global__ __launch_bounds__(kThreads, NB == 4 ? 1 : 2) void int4_decode_kernel(Int4DecodeParams p) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[kWaves][2][kStage];
  constexpr int CH = D == 128 ? 64 : 128;      // keys of a chunk
  constexpr int W = D == 128 ? 1 : 2;          // queries of a block whose scores a lane ends up with
  constexpr int NG = D / kGroup, NDB = D / 16; // column groups, blocks of 16 columns
  constexpr int HV = CH / 64;                  // 64-key halves of a chunk
  constexpr int PROW = 2 * CH + 16;            // bytes of a probability row in LDS (16 more: rows on other banks)
  const int split = blockIdx.x, g = blockIdx.y, v0 = blockIdx.z * kVecs;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int k = lane & 15, a = lane >> 4;
  const int G = p.H / p.Hkv, R = p.T * G - v0 < kVecs ? p.T * G - v0 : kVecs;
  const int64_t n = live_length(p), len = split_keys(n, p.n_splits), begin = split * len;
  const int64_t end = begin + len < n ? begin + len : n;
  const int count = end > begin ? (int)(end - begin) : 0;

  if (p.knew != nullptr && gridDim.z == 1) {
    // the length before clamping places the new rows; those outside the cache are left out
    const int64_t raw = p.n_dev ? *p.n_dev : p.n;
    const int64_t hi = begin + len < p.cap ? begin + len : p.cap;
    if (raw > begin && raw - p.T < hi) {
      append_rows<D>(p, raw, begin, hi, g, tid);
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): the rows are in L2 before any wave of this workgroup reads them
      __syncthreads();
    }
  }
  if (count == 0 && p.n_splits > 1) return;  // no partial: the merge knows the live splits

  // the query operand: fragment i of block b, element 2 m / 2 m + 1 = column 8 i + m / 8 i + m + 4 of the lane's group
  bf16x8_t qa[NB][4];
  f32x4_t qs[NB];  // sums of the queries' groups, where the scores are
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int v = v0 + 4 * b + (k & 3);
    const bool on = (k >> 2) == a && 4 * b + (k & 3) < R;
    const uint16_t* qr = p.q + (on ? (v / G) * p.sq0 + (g * G + v % G) * p.sq1 + kGroup * (D == 128 ? a : a & 1) : 0);
    qs[b] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4_t w = on ? ld16(qr + 8 * i) : u32x4_t{0, 0, 0, 0};
      qa[b][i] = as_bf16x8(u32x4_t{(w[0] & 0xffffu) | (w[2] << 16), (w[0] >> 16) | (w[2] & 0xffff0000u),
                                   (w[1] & 0xffffu) | (w[3] << 16), (w[1] >> 16) | (w[3] & 0xffff0000u)});
      constexpr uint32_t one = F16 ? 0x3c003c00u : 0x3f803f80u;
      qs[b] = mma16<F16>(qa[b][i], as_bf16x8(u32x4_t{one, one, one, one}), qs[b]);
    }
  }

  const int64_t row0 = begin;
  auto rsrc = [&](const void* base, int64_t row_bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(static_cast<const uint8_t*>(base)) + row0 * row_bytes, 0,
                                             (int)(count * row_bytes), 0x00020000);
  };
  const __amdgpu_buffer_rsrc_t kqr = rsrc(p.kq + g * p.skq, D / 2), kpr = rsrc(p.kp + g * p.skp, D / 8);
  const __amdgpu_buffer_rsrc_t vqr = rsrc(p.vq + g * p.svq, D / 2), vpr = rsrc(p.vp + g * p.svp, D / 8);

  // Where lane l's 16 bytes of load i come from (they land at 1024 i + 16 l). Loads cover whole contiguous kilobytes; inside,
  // pieces are placed for the reads below. key(k, u) is the key of lane k in score step u, with
  //   key(k, u) = 16 (k >> 2) + 8 ((k >> 1) & 1) + 4 (u & 1) + 2 (k & 1) + (u >> 1),
  // so that a lane's four steps are four neighbouring elements of the value operand (codes16's order).
  uint32_t koff[2], voff, poff;  // K codes: even and odd loads differ only by a constant xor
  auto unplace = [](int pos) { return ((pos >> 1) & 1) << 3 | (pos >> 3) << 2 | (pos & 1) << 1 | ((pos >> 2) & 1); };
  if constexpr (D == 128) {
    koff[0] = 64 * unplace(lane >> 2) + 16 * (lane & 3);
    koff[1] = 0;
    voff = 64 * (lane >> 2) + 16 * ((lane & 3) ^ (lane >> 4));
    const int kk = lane & 15, u = lane >> 4;  // params: slot 16 u + k holds key(k, u)
    poff = 16 * (16 * (kk >> 2) + 8 * ((kk >> 1) & 1) + 4 * (u & 1) + 2 * (kk & 1) + (u >> 1));
  } else {
    const int pos = (lane >> 1) & 15;
    koff[0] = 512 * (lane >> 5) + 32 * unplace(pos) + 16 * (lane & 1);
    koff[1] = 512 * (lane >> 5) + 32 * unplace(pos ^ 4) + 16 * (lane & 1);
    voff = 512 * (lane >> 5) + 32 * pos + 16 * ((lane & 1) ^ (pos >> 3));
    const int kk = lane & 15, half = (lane >> 4) & 1, u = lane >> 5;  // slot 32 (u & 1) + 16 half + k: keys key(k, u), + 1
    poff = 8 * (64 * half + 16 * (kk >> 2) + 8 * ((kk >> 1) & 1) + 4 * u + 2 * (kk & 1));
  }
  auto fetch = [&](int c, int st) {
    uint8_t* base = sm[wave][st];
    auto ld = [&](__amdgpu_buffer_rsrc_t r, int at, uint32_t off) {
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, reinterpret_cast<lds_void*>(reinterpret_cast<uintptr_t>(base + at)), 16, off, 0, 0, 2 /* non-temporal */);
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t off;
      if constexpr (D == 128) off = koff[0] ^ (16 * (-i & 3));  // the piece's bits are 4 and 5 of the offset
      else off = koff[i & 1];
      ld(kqr, 1024 * i, c * 4096 + 1024 * i + off);
    }
    ld(kpr, kKp, c * 1024 + poff);
#pragma unroll
    for (int i = 0; i < 4; ++i) ld(vqr, kVq + 1024 * i, c * 4096 + 1024 * i + voff);
    ld(vpr, kVp, c * 1024 + poff);
  };
  // where the reads of a stage start
  uint32_t kread[2], kpread, vpread;
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
  const int key_k = (D == 128 ? 0 : 64 * (a >> 1)) + 16 * (k >> 2) + 8 * ((k >> 1) & 1) + 2 * (k & 1);

  // how many of the split's keys each of the lane's queries attends, and the fewest over all
  int lim[NB][W];
#pragma unroll
  for (int b = 0; b < NB; ++b)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int v = v0 + 4 * b + (D == 128 ? a : (a & 1) + 2 * w);
      const int64_t seen = seen_keys(p, n, v / G) - begin;
      lim[b][w] = (int)(seen < 0 ? 0 : seen < count ? seen : count);
    }
  int fewest;
  {
    const int64_t seen = seen_keys(p, n, v0 / G) - begin;
    fewest = (int)(seen < 0 ? 0 : seen < count ? seen : count);
  }

  float m[NB][W], l[NB][W], zs[NB][4];
  f32x4_t o[NB][NDB], ones[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int w = 0; w < W; ++w) { m[b][w] = -1.0e30f; l[b][w] = 0.0f; }
#pragma unroll
    for (int t = 0; t < 4; ++t) zs[b][t] = 0.0f;
    ones[b] = f32x4_t{0, 0, 0, 0};
#pragma unroll
    for (int db = 0; db < NDB; ++db) o[b][db] = f32x4_t{0, 0, 0, 0};
  }

  const int chunks = (count + CH - 1) / CH;
  int st = 0;
  if (wave < chunks) fetch(wave, 0);
  for (int c = wave; c < chunks; c += kWaves, st ^= 1) {
    if (c + kWaves < chunks) {
      fetch(c + kWaves, st ^ 1);
      __builtin_amdgcn_s_waitcnt(0x0F7A);  // vmcnt(10): this chunk's ten loads have landed
    } else {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
    }
    wave_fence();
    uint8_t* s = sm[wave][st];
    const bool whole = (c + 1) * CH <= fewest;
    if constexpr (D == 64) {
      // an odd last key's params share their 16-byte piece with a row past the range: read them apart
      if ((count & 1) && (c + 1) * CH > count && lane < 4) {
        const int key = count - 1 - c * CH, kk = 4 * ((key >> 4) & 3) + 2 * ((key >> 3) & 1) + ((key >> 1) & 1);
        const uint32_t* src = (lane & 2 ? p.vp + g * p.svp : p.kp + g * p.skp) + 2 * (end - 1) + (lane & 1);
        *reinterpret_cast<uint32_t*>(s + (lane & 2 ? kVp : kKp) + 512 * ((key >> 2) & 1) + 256 * (key >> 6) + 16 * kk +
                                     8 * (key & 1) + 4 * (lane & 1)) = *src;
      }
    }
    wave_fence();

    float x[NB][W][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const u32x4_t kw = *reinterpret_cast<const u32x4_t*>(s + kread[u >> 1] + (D == 128 ? 512 : 256) * (u & 1));
      uint32_t kp = *reinterpret_cast<const uint32_t*>(s + kpread + (D == 128 ? 256 * u : 512 * (u & 1) + 8 * (u >> 1)));
      const int key = c * CH + key_k + 4 * (u & 1) + (u >> 1);
      if (!whole) kp = key < count ? kp : 0u;
      const float sc = f16_lo(kp) * p.c, zc = fmaf(-16.0f, f16_lo(kp), f16_hi(kp)) * p.c;
      f32x4_t acc[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[b] = f32x4_t{0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bf16x8_t kf = codes16<F16>(kw[i]);
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] = mma16<F16>(qa[b][i], kf, acc[b]);
      }
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float y[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) y[h] = fmaf(sc, acc[b][h], zc * qs[b][h]);
        if constexpr (D == 128) {
          x[b][0][u] = sum_rows16(sum_rows32(y[0], y[2]), sum_rows32(y[1], y[3]));
        } else {
          x[b][0][u] = sum_rows16(y[0], y[1]);
          x[b][1][u] = sum_rows16(y[2], y[3]);
        }
        if (!whole) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (key >= lim[b][w]) x[b][w][u] = -__builtin_huge_valf();
        }
      }
    }
    float pr[NB][W][4];
    bool over = false;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          pr[b][w][u] = fast_exp2(x[b][w][u] - m[b][w]);
          over |= !(pr[b][w][u] <= kOver);
        }
    if (__builtin_amdgcn_ballot_w64(over)) {
#pragma unroll
      for (int b = 0; b < NB; ++b) {
        float alpha[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
          float mx = row_max(fmaxf(fmaxf(x[b][w][0], x[b][w][1]), fmaxf(x[b][w][2], x[b][w][3])));
          if constexpr (D == 64) mx = xhalf_max(mx);
          const float mn = fmaxf(m[b][w], mx);
          alpha[w] = fast_exp2(m[b][w] - mn);
          m[b][w] = mn;
          l[b][w] *= alpha[w];
#pragma unroll
          for (int u = 0; u < 4; ++u) pr[b][w][u] = fast_exp2(x[b][w][u] - mn);
#pragma unroll
          for (int t = 0; t < NG; ++t) zs[b][NG * w + t] *= alpha[w];
        }
        // column 4 t + h of the sums belongs to query h
        float al[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) al[h] = D == 128 ? lane_value(alpha[0], 16 * h) : lane_value(alpha[W - 1 ? h >> 1 : 0], 16 * (h & 1));
        const float ac = k & 2 ? (k & 1 ? al[3] : al[2]) : (k & 1 ? al[1] : al[0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ones[b][e] *= ac;
#pragma unroll
          for (int db = 0; db < NDB; ++db) o[b][db][e] *= ac;
        }
      }
    }
    // probabilities times V scales, [4 t + h][key] in the space of the K rows, then the operand of every block
    bf16x8_t pb[NB][2 * HV], pl[NB][2 * HV];
    uint32_t vp[4][NG];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int key = c * CH + key_k + 4 * (u & 1) + (u >> 1);
      if constexpr (D == 128) {
        const u32x4_t r = *reinterpret_cast<const u32x4_t*>(s + vpread + 256 * u);
#pragma unroll
        for (int t = 0; t < 4; ++t) vp[u][t] = r[t];
      } else {
        const u32x2_t r = *reinterpret_cast<const u32x2_t*>(s + vpread + 512 * (u & 1) + 8 * (u >> 1));
        vp[u][0] = r[0];
        vp[u][1] = r[1];
      }
      if (!whole) {
#pragma unroll
        for (int t = 0; t < NG; ++t) vp[u][t] = key < count ? vp[u][t] : 0u;
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      wave_fence();
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int u = 0; u < 4; ++u) l[b][w] += pr[b][w][u];
#pragma unroll
        for (int t = 0; t < NG; ++t) {
          float q[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            q[u] = pr[b][w][u] * f16_lo(vp[u][t]);
            // the sums take 24 off every code, so that a rounded probability meets -8..7: z + 8 s here
            zs[b][NG * w + t] = fmaf(pr[b][w][u], f16_hi(vp[u][t]), fmaf(8.0f, q[u], zs[b][NG * w + t]));
          }
          const uint32_t h0 = pack_bf16x2(q[0], q[1]), h1 = pack_bf16x2(q[2], q[3]);
          const int col = D == 128 ? 4 * t + a : 4 * t + (a & 1) + 2 * w;
          uint8_t* dst = s + col * PROW + (D == 128 ? 0 : 128 * (a >> 1)) + 8 * k;
          *reinterpret_cast<u32x2_t*>(dst) = u32x2_t{h0, h1};
          if constexpr (TWO) {
            const uint32_t l0 = pack_bf16x2(q[0] - __uint_as_float(h0 << 16), q[1] - __uint_as_float(h0 & 0xffff0000u));
            const uint32_t l1 = pack_bf16x2(q[2] - __uint_as_float(h1 << 16), q[3] - __uint_as_float(h1 & 0xffff0000u));
            *reinterpret_cast<u32x2_t*>(dst + 4 * NG * PROW) = u32x2_t{l0, l1};
          }
        }
      }
      wave_fence();
      const uint8_t* src = s + (D == 128 ? k : k & 7) * PROW + 32 * a;  // head_dim 64: columns 8..15 repeat and are not used
#pragma unroll
      for (int j = 0; j < 2 * HV; ++j) {
        pb[b][j] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(src + 128 * (j >> 1) + 16 * (j & 1)));
        if constexpr (TWO)
          pl[b][j] = as_bf16x8(*reinterpret_cast<const u32x4_t*>(src + 4 * NG * PROW + 128 * (j >> 1) + 16 * (j & 1)));
      }
    }
    const bf16x8_t one = as_bf16x8(u32x4_t{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u});
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int j = 0; j < 2 * HV; ++j) {
        ones[b] = mma16_bf16(one, pb[b][j], ones[b]);
        if constexpr (TWO) ones[b] = mma16_bf16(one, pl[b][j], ones[b]);
      }
#pragma unroll
    for (int hv = 0; hv < HV; ++hv)
#pragma unroll
      for (int db = 0; db < NDB; ++db) {
        // lane k points at row 16 a + k, 8 bytes of column block db, and gets column k of the 16 rows
        const uint32_t at = D == 128 ? 1024 * a + 64 * k + 16 * ((db >> 1) ^ (k >> 2)) + 8 * (db & 1)
                                     : 2048 * hv + 512 * a + 32 * k + 16 * ((db >> 1) ^ (k >> 3)) + 8 * (db & 1);
        const v2i_t t = __builtin_amdgcn_ds_read_tr4_b64_v2i32(reinterpret_cast<__attribute__((address_space(3))) v2i_t*>(
            reinterpret_cast<uintptr_t>(s + kVq + at)));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bf16x8_t vf = codes16<false>((uint32_t)(j ? t.y : t.x));
#pragma unroll
          for (int b = 0; b < NB; ++b) {
            o[b][db] = mma16_bf16(vf, pb[b][2 * hv + j], o[b][db]);
            if constexpr (TWO) o[b][db] = mma16_bf16(vf, pl[b][2 * hv + j], o[b][db]);
          }
        }
      }
    wave_fence();
  }

  // the wave's state to its own LDS (all of its loads have landed): per vector m, l, the minima's part per group, o
  constexpr int NV = 4 * NB;
  float* mine = reinterpret_cast<float*>(sm[wave]);
  float* const mm = mine, *const ll = mine + NV, *const zz = mine + 2 * NV, *const oo = mine + 2 * NV + NG * NV;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
#pragma unroll
    for (int w = 0; w < W; ++w) {
      float sum = row_sum(l[b][w]);
      if constexpr (D == 64) sum = xhalf_sum(sum);
      const int v = 4 * b + (D == 128 ? a : (a & 1) + 2 * w);
      if (k == 0) {
        mm[v] = m[b][w];
        ll[v] = sum;
      }
#pragma unroll
      for (int t = 0; t < NG; ++t) {
        float z = row_sum(zs[b][NG * w + t]);
        if constexpr (D == 64) z = xhalf_sum(z);
        if (k == 0) zz[NG * v + t] = z;
      }
    }
#pragma unroll
    for (int db = 0; db < NDB; ++db)
      if ((k >> 2) == db / 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) oo[(4 * b + (k & 3)) * D + 16 * db + 4 * a + e] = fmaf(-24.0f, ones[b][e], o[b][db][e]);
      }
  }
  __syncthreads();
  for (int i = tid; i < R * D; i += kThreads) {
    const int r = i / D, d = i % D, v = v0 + r, t = v / G, hd = g * G + v % G;
    float M = -1.0e30f, L = 0.0f, O = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) M = fmaxf(M, reinterpret_cast<const float*>(sm[w])[r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float* f = reinterpret_cast<const float*>(sm[w]);
      const float wt = fast_exp2(f[r] - M);
      L += wt * f[NV + r];
      O += wt * (f[2 * NV + NG * NV + r * D + d] + f[2 * NV + NG * r + d / kGroup]);
    }
    if (p.n_splits == 1) {
      p.out[t * p.so0 + hd * p.so1 + d] = to16<F16>(L > 0.0f ? O / L : 0.0f);
    } else {
      float* dst = p.part + (((int64_t)t * p.H + hd) * p.n_splits + split) * (D + 2);
      dst[d] = O;
      if (d == 0) { dst[D] = M; dst[D + 1] = L; }
    }
  }
}

// The partials of the live splits under one maximum: a workgroup per (query vector, 16 columns), thread (column, lane group)
// folding every 16th split, 8 loaded at a time; the groups then combine through LDS. A row without keys is zero.
constexpr int kMergeCols = 16, kMergeGroups = 16, kMergePer = 8;
template <int D, bool F16>
__global__ __launch_bounds__(kMergeCols * kMergeGroups) void int4_merge_kernel(Int4DecodeParams p) {
  __shared__ float sm_m[kMergeGroups], sm_l[kMergeGroups], sm_o[kMergeGroups][kMergeCols];
  const int v = blockIdx.x, dl = threadIdx.x % kMergeCols, grp = threadIdx.x / kMergeCols, d = kMergeCols * blockIdx.y + dl;
  const int64_t n = live_length(p), len = split_keys(n, p.n_splits);
  const int live = (int)((n + len - 1) / len);
  const float* base = p.part + (int64_t)v * p.n_splits * (D + 2);
  float M = -1.0e30f, L = 0.0f, O = 0.0f;
  for (int i0 = grp; i0 < live; i0 += kMergeGroups * kMergePer) {
    float mv[kMergePer], lv[kMergePer], ov[kMergePer];
#pragma unroll
    for (int i = 0; i < kMergePer; ++i) {
      const int s = i0 + kMergeGroups * i;
      const bool ok = s < live;
      const float* r = base + (int64_t)(ok ? s : 0) * (D + 2);
      mv[i] = ok ? r[D] : -1.0e30f;
      lv[i] = ok ? r[D + 1] : 0.0f;
      ov[i] = ok ? r[d] : 0.0f;
    }
    float mn = M;
#pragma unroll
    for (int i = 0; i < kMergePer; ++i) mn = fmaxf(mn, mv[i]);
    const float al = fast_exp2(M - mn);
    L *= al;
    O *= al;
#pragma unroll
    for (int i = 0; i < kMergePer; ++i) {
      const float w = fast_exp2(mv[i] - mn);
      L += w * lv[i];
      O += w * ov[i];
    }
    M = mn;
  }
  sm_o[grp][dl] = O;
  if (dl == 0) { sm_m[grp] = M; sm_l[grp] = L; }
  __syncthreads();
  if (grp == 0) {
    float mx = sm_m[0];
#pragma unroll
    for (int i = 1; i < kMergeGroups; ++i) mx = fmaxf(mx, sm_m[i]);
    float lt = 0.0f, ot = 0.0f;
#pragma unroll
    for (int i = 0; i < kMergeGroups; ++i) {
      const float w = fast_exp2(sm_m[i] - mx);
      lt += w * sm_l[i];
      ot += w * sm_o[i][dl];
    }
    p.out[(v / p.H) * p.so0 + (v % p.H) * p.so1 + d] = to16<F16>(lt > 0.0f ? ot / lt : 0.0f);
  }
}

// The step's new rows in a launch of their own, where several passes read them.
template <int D>
__global__ __launch_bounds__(kThreads) void int4_append_kernel(Int4DecodeParams p) {
  append_rows<D>(p, p.n_dev ? *p.n_dev : p.n, 0, p.cap, blockIdx.x, threadIdx.x);
}

template <int D, bool F16>
hipError_t launch_decode_t(const Int4DecodeParams& p, hipStream_t stream) {
  const int vecs = p.T * (p.H / p.Hkv), passes = (vecs + kVecs - 1) / kVecs;
  if (p.knew && passes > 1) hipLaunchKernelGGL(int4_append_kernel<D>, dim3(p.Hkv), dim3(kThreads), 0, stream, p);
  const dim3 grid(p.n_splits, p.Hkv, passes);
  if (vecs <= 4) hipLaunchKernelGGL((int4_decode_kernel<D, F16, 1, F16>), grid, dim3(kThreads), 0, stream, p);
  else if (vecs <= 8) hipLaunchKernelGGL((int4_decode_kernel<D, F16, 2, F16>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((int4_decode_kernel<D, F16, 4, F16>), grid, dim3(kThreads), 0, stream, p);
  if (p.n_splits > 1)
    hipLaunchKernelGGL((int4_merge_kernel<D, F16>), dim3(p.T * p.H, D / kMergeCols),
                       dim3(kMergeCols * kMergeGroups), 0, stream, p);
  return hipGetLastError();
}

dim3 row_grid(int D, int heads, int64_t rows, bool two) {
  return dim3((unsigned)((rows + 2048 / D - 1) / (2048 / D)), (unsigned)heads, two ? 2u : 1u);
}

}  // namespace

hipError_t launch_int4_quantize(const Int4Rows& k, const Int4Rows* v, int kind, int heads, int64_t rows, int D,
                                hipStream_t stream) {
  if (rows <= 0 || heads <= 0) return hipSuccess;
  const Int4Set s0{k.x, k.q, k.p, k.sx0, k.sx1, k.sq0, k.sp0};
  const Int4Set s1 = v ? Int4Set{v->x, v->q, v->p, v->sx0, v->sx1, v->sq0, v->sp0} : s0;
  const dim3 grid = row_grid(D, heads, rows, v != nullptr);
  switch (D) {
    case 32: hipLaunchKernelGGL(int4_quantize_kernel<32>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    case 64: hipLaunchKernelGGL(int4_quantize_kernel<64>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    case 128: hipLaunchKernelGGL(int4_quantize_kernel<128>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    case 256: hipLaunchKernelGGL(int4_quantize_kernel<256>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_int4_dequantize(const Int4Rows& k, const Int4Rows* v, int kind, int heads, int64_t rows, int D,
                                  hipStream_t stream) {
  if (rows <= 0 || heads <= 0) return hipSuccess;
  const Int4ReadSet s0{k.q, k.p, const_cast<void*>(k.x), k.sq0, k.sp0};
  const Int4ReadSet s1 = v ? Int4ReadSet{v->q, v->p, const_cast<void*>(v->x), v->sq0, v->sp0} : s0;
  const dim3 grid = row_grid(D, heads, rows, v != nullptr);
  switch (D) {
    case 32: hipLaunchKernelGGL(int4_dequantize_kernel<32>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    case 64: hipLaunchKernelGGL(int4_dequantize_kernel<64>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    case 128: hipLaunchKernelGGL(int4_dequantize_kernel<128>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    case 256: hipLaunchKernelGGL(int4_dequantize_kernel<256>, grid, dim3(256), 0, stream, s0, s1, kind, rows); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_int4_decode(const Int4DecodeParams& p, hipStream_t stream) {
  if (p.D == 64) return p.f16 ? launch_decode_t<64, true>(p, stream) : launch_decode_t<64, false>(p, stream);
  return p.f16 ? launch_decode_t<128, true>(p, stream) : launch_decode_t<128, false>(p, stream);
}

}  // namespace bb
