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
// Attention over the packed rows, split over the keys. Workgroup (split, KV head, pass): the pass's up to 16 query
// vectors (token-major, T tokens x G heads of the KV head) against the split's keys. The length comes from device memory
// when n_dev is set, so every launch shape depends on host values alone.
constexpr int kVecs = 16;
constexpr int kTile = 256;

BB_DEV int64_t live_length(const Int4DecodeParams& p) {
  int64_t n = p.n_dev ? *p.n_dev : p.n;
  return n < 0 ? 0 : n > p.cap ? p.cap : n;
}
BB_DEV int64_t split_keys(int64_t n, int n_splits) {
  int64_t len = (n + n_splits - 1) / n_splits;
  len = (len + 15) & ~(int64_t)15;
  return len < kInt4MinSplit ? kInt4MinSplit : len;
}
// Keys that token t of T attends.
BB_DEV int64_t seen_keys(const Int4DecodeParams& p, int64_t n, int t) { return p.causal ? n - p.T + 1 + t : n; }

template <int D, bool F16>
__global__ __launch_bounds__(kTile) void int4_decode_kernel(Int4DecodeParams p) {
  __shared__ float sq[kVecs][D], sx[kVecs][kTile], sm[kVecs], sl[kVecs], red[4];
  const int split = blockIdx.x, g = blockIdx.y, v0 = blockIdx.z * kVecs, tid = threadIdx.x;
  const int G = p.H / p.Hkv, R = p.T * G - v0 < kVecs ? p.T * G - v0 : kVecs;
  const int64_t n = live_length(p), len = split_keys(n, p.n_splits), begin = split * len;
  const int64_t end = begin + len < n ? begin + len : n;
  if (begin >= n) return;
  for (int i = tid; i < R * D; i += kTile) {
    const int v = v0 + i / D;
    const uint16_t h = p.q[(v / G) * p.sq0 + (g * G + v % G) * p.sq1 + i % D];
    sq[i / D][i % D] = F16 ? (float)__builtin_bit_cast(_Float16, h) : bf16_to_f32(h);
  }
  if (tid < kVecs) { sm[tid] = -1.0e30f; sl[tid] = 0.0f; }
  const uint8_t* kq = p.kq + g * p.skq;
  const uint8_t* vq = p.vq + g * p.svq;
  const uint32_t* kp = p.kp + g * p.skp;
  const uint32_t* vp = p.vp + g * p.svp;
  float o[kVecs];
#pragma unroll
  for (int r = 0; r < kVecs; ++r) o[r] = 0.0f;
  for (int64_t j0 = begin; j0 < end; j0 += kTile) {
    __syncthreads();
    const int64_t j = j0 + tid;
    for (int r = 0; r < R; ++r) {
      float x = -__builtin_huge_valf();
      if (j < end && j < seen_keys(p, n, (v0 + r) / G)) {
        x = 0.0f;
        for (int gr = 0; gr < D / kGroup; ++gr) {
          const uint32_t pr = kp[j * (D / kGroup) + gr];
          const float s = f16_lo(pr), z = f16_hi(pr);
          for (int w4 = 0; w4 < 4; ++w4) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(kq + j * (D / 2) + 16 * gr + 4 * w4);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              x = fmaf(fmaf(s, (float)((w >> (4 * i)) & 15u), z), sq[r][32 * gr + 8 * w4 + i], x);
          }
        }
        x *= p.c;
      }
      sx[r][tid] = x;
    }
    __syncthreads();
    for (int r = 0; r < R; ++r) {
      float t = sx[r][tid];
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) t = fmaxf(t, __shfl_xor(t, off));
      if ((tid & 63) == 0) red[tid >> 6] = t;
      __syncthreads();
      const float mn = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), sm[r]);
      const float a = fast_exp2(sm[r] - mn);
      const float e = fast_exp2(sx[r][tid] - mn);
      float sum = e;
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
      __syncthreads();
      if ((tid & 63) == 0) red[tid >> 6] = sum;
      sx[r][tid] = e;
      o[r] *= a;
      __syncthreads();
      if (tid == 0) {
        sm[r] = mn;
        sl[r] = sl[r] * a + red[0] + red[1] + red[2] + red[3];
      }
      __syncthreads();
    }
    if (tid < D) {
      const int64_t m = end - j0 < kTile ? end - j0 : kTile;
      for (int i = 0; i < m; ++i) {
        const int64_t jj = j0 + i;
        const uint32_t pr = vp[jj * (D / kGroup) + tid / kGroup];
        const uint32_t b = vq[jj * (D / 2) + tid / 2] >> (4 * (tid & 1));
        const float val = fmaf(f16_lo(pr), (float)(b & 15u), f16_hi(pr));
#pragma unroll
        for (int r = 0; r < kVecs; ++r)
          if (r < R) o[r] = fmaf(sx[r][i], val, o[r]);
      }
    }
  }
  __syncthreads();
  for (int r = 0; r < R; ++r) {
    const int v = v0 + r;
    float* dst = p.part + (((int64_t)(v / G) * p.H + g * G + v % G) * p.n_splits + split) * (D + 2);
    if (tid < D) dst[tid] = o[r];
    if (tid == 0) { dst[D] = sm[r]; dst[D + 1] = sl[r]; }
  }
}

// One workgroup per query vector: the live splits' partials under one maximum. A row without keys is zero.
template <int D, bool F16>
__global__ __launch_bounds__(D) void int4_merge_kernel(Int4DecodeParams p) {
  const int64_t n = live_length(p), len = split_keys(n, p.n_splits);
  const int live = (int)((n + len - 1) / len), v = blockIdx.x, d = threadIdx.x;
  const float* base = p.part + (int64_t)v * p.n_splits * (D + 2);
  float M = -1.0e30f, L = 0.0f, O = 0.0f;
  for (int s = 0; s < live; ++s) M = fmaxf(M, base[s * (D + 2) + D]);
  for (int s = 0; s < live; ++s) {
    const float w = fast_exp2(base[s * (D + 2) + D] - M);
    L += w * base[s * (D + 2) + D + 1];
    O += w * base[s * (D + 2) + d];
  }
  p.out[(v / p.H) * p.so0 + (v % p.H) * p.so1 + d] = to16<F16>(L > 0.0f ? O / L : 0.0f);
}

// The step's new rows into cache rows n - T .. n - 1 (rows outside the cache are left out).
template <int D>
__global__ __launch_bounds__(256) void int4_append_kernel(Int4DecodeParams p) {
  constexpr int LPR = D / 8;
  const int t = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, c = threadIdx.x % LPR, g = blockIdx.y;
  if (t >= p.T) return;
  const int64_t n = p.n_dev ? *p.n_dev : p.n, row = n - p.T + t;
  if (row < 0 || row >= p.cap) return;
  const bool vt = blockIdx.z;
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

template <int D, bool F16>
hipError_t launch_decode_t(const Int4DecodeParams& p, hipStream_t stream) {
  if (p.knew)
    hipLaunchKernelGGL(int4_append_kernel<D>, dim3((p.T + 2048 / D - 1) / (2048 / D), p.Hkv, 2), dim3(256), 0, stream, p);
  const int passes = (p.T * (p.H / p.Hkv) + kVecs - 1) / kVecs;
  hipLaunchKernelGGL((int4_decode_kernel<D, F16>), dim3(p.n_splits, p.Hkv, passes), dim3(kTile), 0, stream, p);
  hipLaunchKernelGGL((int4_merge_kernel<D, F16>), dim3(p.T * p.H), dim3(D), 0, stream, p);
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
