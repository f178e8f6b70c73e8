// Rotary positions (fa_rotary) and appends to a paged K/V cache (fa_paged_append).
//
// Pair i of a head row at position p turns by 2 pi p f_i:
//     (a, b) -> magnitude * (a cos - b sin, b cos + a sin).
// Both kernels read every element once and write it once, so HBM bandwidth bounds them (and
// the launch, for a single token).  The angle is reduced in integers: f_i comes as 64-bit fixed
// point in turns, so p * f_i mod 2^64 is the exact phase of any 32-bit position (a product in
// fp32 is off by 0.06 rad at position 2^20), and its top 32 bits become the reduced angle.
//
// Measured (bf16, D 128, 32 + 8 heads): rotation of 2 x 8192 tokens with its gradient 111 us,
// 6.1 TB/s; one token each of 64 sequences 2.3 us, the launch.  Append of eight prompts of up to
// 2048 tokens to 8-bit pages with q's rotation 59 us (3.6 TB/s; 34 us with 8 + 8 heads): two thirds of the
// issue slots, and a team's chain of lengths, rows, largest magnitude and stores.  One token each of 64
// sequences 3.9 us.
//
// A thread owns a unit of 16 elements of a row: 8 + 8 elements rotary_dim / 2 apart for the half
// layout, 16 neighbours for interleaved pairs and for the copied tail.  It computes the 8 cosines
// and sines of its pairs once and reuses them for several heads of the same token.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>

#include "fa_common.cuh"
#include "fa_internal.h"
#include "flexattn.h"

namespace fa {
namespace {

constexpr int kScaleFloor = -100;  // least exponent of a page's scale

// ------------------------------------------------------------------ elements
// Eight elements as they lie in memory (16 or 32 bytes), and as floats.  Streaming loads: nothing
// is read twice.
template <typename T> struct Io;
template <> struct Io<__nv_bfloat16> {
  struct Raw { uint4 v; };
  static __device__ __forceinline__ Raw fetch(const __nv_bfloat16* p) {
    return {__ldcs(reinterpret_cast<const uint4*>(p))};
  }
  static __device__ __forceinline__ Raw gather(const __nv_bfloat16* p) {  // any alignment
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    return {make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16, h[4] | (uint32_t)h[5] << 16,
                       h[6] | (uint32_t)h[7] << 16)};
  }
  static __device__ __forceinline__ void floats(const Raw& r, float (&f)[8]) {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
};
template <> struct Io<float> {
  struct Raw { float4 a, b; };
  static __device__ __forceinline__ Raw fetch(const float* p) {
    return {__ldcs(reinterpret_cast<const float4*>(p)), __ldcs(reinterpret_cast<const float4*>(p) + 1)};
  }
  static __device__ __forceinline__ Raw gather(const float* p) {
    return {make_float4(p[0], p[1], p[2], p[3]), make_float4(p[4], p[5], p[6], p[7])};
  }
  static __device__ __forceinline__ void floats(const Raw& r, float (&f)[8]) {
    f[0] = r.a.x; f[1] = r.a.y; f[2] = r.a.z; f[3] = r.a.w;
    f[4] = r.b.x; f[5] = r.b.y; f[6] = r.b.z; f[7] = r.b.w;
  }
  static __device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
  static __device__ __forceinline__ float get(const float* p) { return *p; }
  static __device__ __forceinline__ void put(float* p, float x) { *p = x; }
};
// cos and sin of pair i at position pos, times the magnitude.  fp32 tensors get sincospi (2 ulp); for
// bf16 results the special-function unit's sine and cosine of the reduced angle (2^-21 on [-pi, pi])
// lie as far below the rounding of the result, at a fifth of the instructions.
template <typename T>
__device__ __forceinline__ void pair_turn(const FaRotarySpec& r, int i, int pos, float sign, float* c, float* s) {
  const uint64_t phase = (uint64_t)(int64_t)pos * __ldg(r.turns + i);
  const float half_turns = (float)(int32_t)(phase >> 32) * 4.656612873077393e-10f;  // 2^-31: in [-1, 1]
  float sn, cs;
  if constexpr (sizeof(T) == 4) {
    sincospif(half_turns, &sn, &cs);
  } else {
    __sincosf(half_turns * 3.14159265358979f, &sn, &cs);
  }
  *c = cs * r.magnitude;
  *s = sn * (r.magnitude * sign);
}

// Two fp32 values at once: the packed instructions do both at the cost of one.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t x, float* a, float* b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*a), "=f"(*b) : "l"(x));
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t both(float x) { return pack2(x, x); }

// The same for pairs i and i + 1 at a position >= 0, to 2^-23: for keys that are rounded to 8 bits,
// where the special-function unit's error puts more of them on the wrong side of a border (68 of 16 M
// codes against 15; cosines and sines rounded from 64 bits: 12).  The angle is reduced to the nearest
// quarter turn, exactly; then the Taylor series of |y| <= pi / 4, whose first terms left out are
// y^11 / 11! = 2^-29 and y^10 / 10! = 2^-25.  It costs eight prompts of 2048 tokens 3 us (11
// without the packed instructions).
__device__ __forceinline__ void pair_turns(const FaRotarySpec& r, int i, uint32_t pos, float* c, float* s) {
  uint32_t w[2];  // phase + 1/8: its two upper bits are the quarter, the others the angle from its middle
  float yf[2], snf[2], csf[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint64_t turns = __ldg(r.turns + i + k);
    const uint32_t phase = __umulhi(pos, (uint32_t)turns) + pos * (uint32_t)(turns >> 32);
    w[k] = phase + 0x20000000u;
    yf[k] = (float)((int32_t)(w[k] & 0x3fffffffu) - 0x20000000) * 1.4629180792671596e-9f;  // 2 pi / 2^32
  }
  const uint64_t y = pack2(yf[0], yf[1]), z = mul2(y, y);
  uint64_t sn = fma2(z, both(1.f / 362880), both(-1.f / 5040)), cs = fma2(z, both(1.f / 40320), both(-1.f / 720));
  sn = fma2(z, sn, both(1.f / 120));
  cs = fma2(z, cs, both(1.f / 24));
  sn = fma2(z, sn, both(-1.f / 6));
  cs = fma2(z, cs, both(-0.5f));
  sn = mul2(fma2(mul2(y, z), sn, y), both(r.magnitude));
  cs = mul2(fma2(z, cs, both(1.f)), both(r.magnitude));
  unpack2(sn, &snf[0], &snf[1]);
  unpack2(cs, &csf[0], &csf[1]);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const bool odd = w[k] & 0x40000000u;  // negative: the cosine in quarters 1 and 2, the sine in 2 and 3
    c[k] = __uint_as_float(__float_as_uint(odd ? snf[k] : csf[k]) ^ ((w[k] + 0x40000000u) & 0x80000000u));
    s[k] = __uint_as_float(__float_as_uint(odd ? csf[k] : snf[k]) ^ (w[k] & 0x80000000u));
  }
}

// Elements [e0, e0 + 8) and [e1, e1 + 8) of unit u; returns whether the unit is rotated.
__device__ __forceinline__ bool unit_span(const FaRotarySpec& r, int u, int* e0, int* e1) {
  const bool rot = u * 16 < r.rotary_dim;
  const bool half = rot && r.layout == FA_ROTARY_HALF;
  *e0 = half ? 8 * u : 16 * u;
  *e1 = half ? r.rotary_dim / 2 + 8 * u : 16 * u + 8;
  return rot;
}

__device__ __forceinline__ void turn16(float (&g0)[8], float (&g1)[8], const float (&c)[8], const float (&s)[8],
                                       bool inter) {
  if (inter) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a0 = g0[2 * j], b0 = g0[2 * j + 1], a1 = g1[2 * j], b1 = g1[2 * j + 1];
      g0[2 * j] = a0 * c[j] - b0 * s[j];
      g0[2 * j + 1] = b0 * c[j] + a0 * s[j];
      g1[2 * j] = a1 * c[4 + j] - b1 * s[4 + j];
      g1[2 * j + 1] = b1 * c[4 + j] + a1 * s[4 + j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = g0[j], b = g1[j];
      g0[j] = a * c[j] - b * s[j];
      g1[j] = b * c[j] + a * s[j];
    }
  }
}

// ------------------------------------------------------------------ fa_rotary
struct RotaryArgs {
  int B, H, Hkv, T, D, units, heads_per_thread, q_chunks;
  FaTensor q, k, q_out, k_out;
  const int32_t* positions;
  int64_t pos_stride_b;
  int pos_offset;
  float sign;  // -1 turns back
  FaRotarySpec r;
};

// Address of row (b, t) of head h, h counted through q's heads and then k's.
template <typename T>
__device__ __forceinline__ T* head_row(const FaTensor& q, const FaTensor& k, int H, int h, int b, int t) {
  const FaTensor& x = h < H ? q : k;
  return reinterpret_cast<T*>(x.ptr) + (int64_t)b * x.stride_b + (int64_t)(h < H ? h : h - H) * x.stride_h +
         (int64_t)t * x.stride_t;
}

template <typename T>
__device__ __forceinline__ T* row_of(const FaTensor& x, int b, int h, int t) {
  return reinterpret_cast<T*>(x.ptr) + (int64_t)b * x.stride_b + (int64_t)h * x.stride_h + (int64_t)t * x.stride_t;
}

// Heads [h0, h1) of one unit of one token of one tensor.  UN heads are in work and the next UN on their
// way, as they lie in memory: few registers, so that many warps share an SM.
template <typename T, int UN>
__device__ __forceinline__ void rotate_heads(const FaTensor& in, const FaTensor& out, const FaRotarySpec& r, int h0,
                                             int h1, int b, int t, int u, int pos, float sign) {
  int e0, e1;
  const bool rot = unit_span(r, u, &e0, &e1);
  const bool inter = r.layout == FA_ROTARY_INTERLEAVED;
  const int apart = e1 - e0;
  typename Io<T>::Raw raw[UN][2];
  const T* x = row_of<const T>(in, b, h0, t) + e0;
  T* y = row_of<T>(out, b, h0, t) + e0;
  auto fetch = [&](int h) {
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      if (h + i < h1) {
        raw[i][0] = Io<T>::fetch(x);
        raw[i][1] = Io<T>::fetch(x + apart);
      }
      x += in.stride_h;
    }
  };
  fetch(h0);
  float c[8], s[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    c[j] = 1.f;
    s[j] = 0.f;
    if (rot) pair_turn<T>(r, 8 * u + j, pos, sign, &c[j], &s[j]);  // behind the first loads, which it overlaps
  }
#pragma unroll 1
  for (int h = h0; h < h1; h += UN) {
    typename Io<T>::Raw now[UN][2];
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      now[i][0] = raw[i][0];
      now[i][1] = raw[i][1];
    }
    fetch(h + UN);
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      if (h + i < h1) {
        float g0[8], g1[8];
        Io<T>::floats(now[i][0], g0);
        Io<T>::floats(now[i][1], g1);
        if (rot) turn16(g0, g1, c, s, inter);
        Io<T>::store8(y, g0);
        Io<T>::store8(y + apart, g1);
      }
      y += out.stride_h;
    }
  }
}

// blockIdx.y: chunks of q's heads, then of k's.
template <typename T>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a) {
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= (unsigned)a.B * a.T * a.units) return;
  const unsigned tok = idx / a.units, b = tok / a.T;
  const int u = idx % a.units, t = tok % a.T;
  const int pos = a.positions ? __ldg(a.positions + (int64_t)b * a.pos_stride_b + t) : a.pos_offset + t;
  const bool of_k = (int)blockIdx.y >= a.q_chunks;
  const int h0 = ((int)blockIdx.y - (of_k ? a.q_chunks : 0)) * a.heads_per_thread;
  const int h1 = min(h0 + a.heads_per_thread, of_k ? a.Hkv : a.H);
  rotate_heads<T, sizeof(T) == 4 ? 1 : 2>(of_k ? a.k : a.q, of_k ? a.k_out : a.q_out, a.r, h0, h1, b, t, u, pos, a.sign);
}

// Any even rotary_dim, head dim, stride and alignment: a thread owns one pair, or two copied
// elements, of a token for heads_per_thread heads.
template <typename T>
__global__ void __launch_bounds__(256) rotary_pair_kernel(const RotaryArgs a) {
  const unsigned idx = blockIdx.x * 256u + threadIdx.x;
  if (idx >= (unsigned)a.B * a.T * a.units) return;
  const unsigned tok = idx / a.units, b = tok / a.T;
  const int u = idx % a.units, t = tok % a.T, half = a.r.rotary_dim / 2;
  const int pos = a.positions ? __ldg(a.positions + (int64_t)b * a.pos_stride_b + t) : a.pos_offset + t;
  const bool rot = u < half, inter = a.r.layout == FA_ROTARY_INTERLEAVED;
  const int e0 = rot && !inter ? u : 2 * u, e1 = rot && !inter ? half + u : 2 * u + 1;
  float c = 1.f, s = 0.f;
  if (rot) pair_turn<T>(a.r, u, pos, a.sign, &c, &s);
  const int h0 = blockIdx.y * a.heads_per_thread, h1 = min(h0 + a.heads_per_thread, a.H + a.Hkv);
  for (int h = h0; h < h1; ++h) {
    const T* x = head_row<const T>(a.q, a.k, a.H, h, b, t);
    T* y = head_row<T>(a.q_out, a.k_out, a.H, h, b, t);
    const float v0 = Io<T>::get(x + e0), v1 = e1 < a.D ? Io<T>::get(x + e1) : 0.f;
    Io<T>::put(y + e0, rot ? v0 * c - v1 * s : v0);
    if (e1 < a.D) Io<T>::put(y + e1, rot ? v1 * c + v0 * s : v1);
  }
}

// ------------------------------------------------------------------ fa_paged_append
struct AppendArgs {
  int B, H, T, Hkv, D, ps, num_pages, cols, units, pages_per_seq;
  int kv_blocks, q_blocks, heads_per_thread, vec;
  int64_t table_stride;
  FaTensor q, k, v, q_out, kc, vc;
  float *k_scale, *v_scale;
  const int32_t *kv_lens, *new_lens, *table;
  FaRotarySpec r;
  int* status;
};

// The span of new positions [*start, *len) of sequence b, none where the batch has an empty slot; false (and a
// status) when its lengths are out of range.
__device__ __forceinline__ bool new_span(const AppendArgs& a, int b, int* start, int* len) {
  const int n = __ldg(a.kv_lens + b), t = a.new_lens ? __ldg(a.new_lens + b) : n == 0 ? 0 : a.T;
  *start = n - t;
  *len = n;
  const bool ok = t >= 0 && t <= a.T && n >= t && n <= a.cols * a.ps;
  if (!ok) report_status(a.status, FA_ERR_INVALID);
  return ok;
}

__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ uint2 to_e4m3x8(const float (&f)[8], float inv) {
  return make_uint2(to_e4m3x2(f[0] * inv, f[1] * inv) | (to_e4m3x2(f[2] * inv, f[3] * inv) << 16),
                    to_e4m3x2(f[4] * inv, f[5] * inv) | (to_e4m3x2(f[6] * inv, f[7] * inv) << 16));
}

// 2^e with the least e >= kScaleFloor such that top <= 448 * 2^e (448 = 1.75 * 2^8), from top's bits.
__device__ __forceinline__ float page_scale(float top) {
  const uint32_t w = __float_as_uint(top);
  const int e = (int)(w >> 23) - 127 - 8 + ((w & 0x7fffffu) > 0x600000u);
  return __uint_as_float((uint32_t)(max(e, kScaleFloor) + 127) << 23);
}

// One team (a warp, or the block) takes the rows of one (sequence, touched page, K/V head) of K
// or of V.  Its new rows stay in registers as they lie in memory between the search for the largest
// magnitude and the store, so they are read once; teams share nothing, and no atomic decides a value.
// A key's turned values, fp32, wait in shared memory, where each thread reads what it wrote itself (in
// registers, half as many teams would share an SM; turned twice, eight prompts with as many heads of q as
// of K took 45 us, then 37; a warp's team, of few rows, turns them twice).  The page's number and its
// scale are fetched behind the rows' loads.
// PASSES: row groups that a team holds, 16 values a thread each.
template <typename T, bool E4M3, bool WARP, int PASSES>
__device__ __forceinline__ void append_team(const AppendArgs& a, int team, int tid, int nt, int* red, float4* stash) {
  const int which = team & 1, hk = (team >> 1) % a.Hkv, bp = (team >> 1) / a.Hkv;
  const int b = bp / a.pages_per_seq;
  int start, len;
  if (!new_span(a, b, &start, &len)) return;
  const int col = start / a.ps + bp % a.pages_per_seq;
  const int first = col * a.ps;  // position of the page's row 0
  if (first >= len || start == len) return;
  const int page = __ldg(a.table + (int64_t)b * a.table_stride + col);
  const int r0 = max(start - first, 0), r1 = min(len - first, a.ps);  // rows the new tokens take
  const int u = tid % a.units, rows_at_once = nt / a.units, row_in = tid / a.units;
  int e0, e1;
  const bool rot = unit_span(a.r, u, &e0, &e1) && which == 0;
  const bool inter = a.r.layout == FA_ROTARY_INTERLEAVED;
  const FaTensor& x = which ? a.v : a.k;
  const FaTensor& cache = which ? a.vc : a.kc;
  const T* src = reinterpret_cast<const T*>(x.ptr) + (int64_t)b * x.stride_b + (int64_t)hk * x.stride_h;

  typename Io<T>::Raw raw[PASSES][2];
#pragma unroll
  for (int p = 0; p < PASSES; ++p) {
    const int row = r0 + p * rows_at_once + row_in;
    if (row_in < rows_at_once && row < r1) {
      const T* s = src + (int64_t)(first + row - start) * x.stride_t;
      raw[p][0] = a.vec ? Io<T>::fetch(s + e0) : Io<T>::gather(s + e0);
      raw[p][1] = a.vec ? Io<T>::fetch(s + e1) : Io<T>::gather(s + e1);
    }
  }
  const bool known = (unsigned)page < (unsigned)a.num_pages;
  float* scale = (which ? a.v_scale : a.k_scale) + (int64_t)page * a.Hkv + hk;
  const float was = E4M3 && known ? *scale : 0.f;  // read by every thread before the barrier, written after it
  if (!known) {  // the same page for the whole team
    if (tid == 0) report_status(a.status, FA_ERR_INVALID);
    return;
  }
  const int64_t base = (int64_t)page * cache.stride_b + (int64_t)hk * cache.stride_h;
  auto values = [&](int p, float (&g0)[8], float (&g1)[8]) {  // of this thread's row of pass p
    Io<T>::floats(raw[p][0], g0);
    Io<T>::floats(raw[p][1], g1);
    if (rot) {
      const int pos = first + r0 + p * rows_at_once + row_in;
      float c[8], s[8];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        if constexpr (E4M3 && sizeof(T) == 2) {
          pair_turns(a.r, 8 * u + j, pos, &c[j], &s[j]);
        } else {
          pair_turn<T>(a.r, 8 * u + j, pos, 1.f, &c[j], &s[j]);
          pair_turn<T>(a.r, 8 * u + j + 1, pos, 1.f, &c[j + 1], &s[j + 1]);
        }
      }
      turn16(g0, g1, c, s, inter);
    }
  };
  if constexpr (!E4M3) {
    __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(cache.ptr) + base;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int row = r0 + p * rows_at_once + row_in;
      if (row_in < rows_at_once && row < r1) {
        float g0[8], g1[8];
        values(p, g0, g1);
        Io<__nv_bfloat16>::store8(dst + (int64_t)row * cache.stride_t + e0, g0);
        Io<__nv_bfloat16>::store8(dst + (int64_t)row * cache.stride_t + e1, g1);
      }
    }
  } else {
    // The largest finite magnitude, as integers: fp32 or bf16 bits without the sign, plus one step of the
    // exponent, which makes infinities and NaN negative.
    constexpr int kStep = 0x00800000;
    int most = kStep;
    uint32_t most2 = 0x00800080u;  // bf16 values that are not turned: two at once
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int row = r0 + p * rows_at_once + row_in;
      if (row_in < rows_at_once && row < r1) {
        if (sizeof(T) == 2 && !rot) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&raw[p][i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) most2 = __viaddmax_s16x2(w[j] & 0x7fff7fffu, 0x00800080u, most2);
          }
          continue;
        }
        float g0[8], g1[8];
        values(p, g0, g1);
        if constexpr (!WARP) {
          if (rot) {
#pragma unroll
            for (int j = 0; j < 8; j += 4) {
              stash[(4 * p + j / 4) * nt + tid] = make_float4(g0[j], g0[j + 1], g0[j + 2], g0[j + 3]);
              stash[(4 * p + 2 + j / 4) * nt + tid] = make_float4(g1[j], g1[j + 1], g1[j + 2], g1[j + 3]);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          most = __viaddmax_s32(__float_as_int(g0[j]) & 0x7fffffff, kStep, most);
          most = __viaddmax_s32(__float_as_int(g1[j]) & 0x7fffffff, kStep, most);
        }
      }
    }
    most = max(most, max((int)(most2 << 16), (int)(most2 & 0xffff0000u)));
    most = __reduce_max_sync(0xffffffffu, most);
    if constexpr (!WARP) {
      if ((tid & 31) == 0) red[tid >> 5] = most;
      __syncthreads();
      for (int w = 0; w < nt / 32; ++w) most = max(most, red[w]);
    } else {
      __syncwarp();
    }
    const float top = __int_as_float(most - kStep);
    float s = page_scale(top);
    if (r0 > 0) s = fmaxf(s, was);  // rows of the sequence are held: the scale only grows
    uint8_t* dst = reinterpret_cast<uint8_t*>(cache.ptr) + base;
    if (r0 > 0 && s > was) {  // requantise them: exact but for what falls below the smallest step
      const float ratio = was / s;
      const int chunks = a.D / 16;
#pragma unroll 1
      for (int e = tid; e < r0 * chunks; e += nt) {
        uint4* w = reinterpret_cast<uint4*>(dst + (int64_t)(e / chunks) * cache.stride_t + (e % chunks) * 16);
        uint4 v = *w;
        uint32_t* vw = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 lo = from_e4m3x2(vw[i] & 0xffffu), hi = from_e4m3x2(vw[i] >> 16);
          vw[i] = to_e4m3x2(lo.x * ratio, lo.y * ratio) | (to_e4m3x2(hi.x * ratio, hi.y * ratio) << 16);
        }
        *w = v;
      }
    }
    const float inv = 1.f / s;
#pragma unroll
    for (int p = 0; p < PASSES; ++p) {
      const int row = r0 + p * rows_at_once + row_in;
      if (row_in < rows_at_once && row < r1) {
        float g0[8], g1[8];
        if (WARP || !rot) {
          values(p, g0, g1);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j += 4) {
            const float4 w0 = stash[(4 * p + j / 4) * nt + tid], w1 = stash[(4 * p + 2 + j / 4) * nt + tid];
            g0[j] = w0.x, g0[j + 1] = w0.y, g0[j + 2] = w0.z, g0[j + 3] = w0.w;
            g1[j] = w1.x, g1[j + 1] = w1.y, g1[j + 2] = w1.z, g1[j + 3] = w1.w;
          }
        }
        uint8_t* d = dst + (int64_t)row * cache.stride_t;
        *reinterpret_cast<uint2*>(d + e0) = to_e4m3x8(g0, inv);
        *reinterpret_cast<uint2*>(d + e1) = to_e4m3x8(g1, inv);
      }
    }
    if (tid == 0 && s != was) *scale = s;
  }
}

// kv_blocks blocks append and the rest rotate q, spread evenly over the grid: appends wait for memory
// most of the time, and q's stream of loads and stores fills it.
// NT: the most threads a block may have.
template <typename T, bool E4M3, bool WARP, int PASSES, int NT>
__global__ void __launch_bounds__(NT, (NT == 512 || sizeof(T) == 4 ? 512 : PASSES == 4 ? 768 : 1024) / NT) append_kernel(const AppendArgs a) {
  __shared__ int red[16];
  extern __shared__ float4 stash[];  // blocks that append 8-bit rows: 4 x PASSES a thread
  const int before = (int)((int64_t)blockIdx.x * a.kv_blocks / gridDim.x);  // appending blocks before this one
  if ((int)((int64_t)(blockIdx.x + 1) * a.kv_blocks / gridDim.x) > before) {
    const int teams = a.B * a.pages_per_seq * a.Hkv * 2;
    if constexpr (WARP) {
      const int team = before * 4 + (threadIdx.x >> 5);
      if (team < teams) append_team<T, E4M3, true, PASSES>(a, team, threadIdx.x & 31, 32, red, stash);
    } else {
      append_team<T, E4M3, false, PASSES>(a, before, threadIdx.x, blockDim.x, red, stash);
    }
    return;
  }
  const unsigned qb = blockIdx.x - before;  // (token block, head chunk), head chunk outermost
  const unsigned idx = (qb % a.q_blocks) * blockDim.x + threadIdx.x;
  if (idx >= (unsigned)a.B * a.T * a.units) return;
  const unsigned tok = idx / a.units, b = tok / a.T;
  const int u = idx % a.units, t = tok % a.T;
  const int h0 = (qb / a.q_blocks) * a.heads_per_thread, h1 = min(h0 + a.heads_per_thread, a.H);
  int start, len;
  const bool ok = new_span(a, b, &start, &len);
  if (ok && start + t < len && a.vec) {
    rotate_heads<T, sizeof(T) == 4 || PASSES == 2 ? 1 : 2>(a.q, a.q_out, a.r, h0, h1, b, t, u, start + t, 1.f);
    return;
  }
  int e0, e1;
  const bool rot = unit_span(a.r, u, &e0, &e1);
  float c[8], s[8];
  if (ok && start + t < len && rot) {
#pragma unroll
    for (int j = 0; j < 8; ++j) pair_turn<T>(a.r, 8 * u + j, start + t, 1.f, &c[j], &s[j]);
  }
  for (int h = h0; h < h1; ++h) {  // padding rows, and tensors that 16-byte accesses do not fit
    float g0[8] = {0.f}, g1[8] = {0.f};
    if (ok && start + t < len) {
      const T* x = row_of<const T>(a.q, b, h, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        g0[j] = Io<T>::get(x + e0 + j);
        g1[j] = Io<T>::get(x + e1 + j);
      }
      if (rot) turn16(g0, g1, c, s, a.r.layout == FA_ROTARY_INTERLEAVED);
    }
    T* y = row_of<T>(a.q_out, b, h, t);
    if (a.vec) {
      Io<T>::store8(y + e0, g0);
      Io<T>::store8(y + e1, g1);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        Io<T>::put(y + e0 + j, g0[j]);
        Io<T>::put(y + e1 + j, g1[j]);
      }
    }
  }
}

// Heads a thread takes: its cosines and sines serve all of them, but the grid should still fill
// the SMs (148 x 512 threads, a quarter of what they hold), and a single token spreads over as many threads as it has heads.
int heads_per_thread(int64_t token_units, int heads) {
  int n = 1;
  while (n < 8 && token_units * ((heads + 2 * n - 1) / (2 * n)) >= 148 * 512) n *= 2;
  return n;
}

bool vec_ok(const FaTensor& t, int es) {
  return (reinterpret_cast<uintptr_t>(t.ptr) & 15u) == 0 && (t.stride_b * es) % 16 == 0 && (t.stride_h * es) % 16 == 0 &&
         (t.stride_t * es) % 16 == 0;
}

int check_spec(const FaRotarySpec& r, int D, const char* who) {
  char msg[160];
  if (r.rotary_dim < 0 || r.rotary_dim > D || r.rotary_dim % 2) {
    snprintf(msg, sizeof(msg), "%s: rotary_dim %d (need an even number up to the head dim %d)", who, r.rotary_dim, D);
    return set_last_error(FA_ERR_INVALID, msg);
  }
  if (r.layout != FA_ROTARY_HALF && r.layout != FA_ROTARY_INTERLEAVED) {
    snprintf(msg, sizeof(msg), "%s: unknown rotary layout %d", who, r.layout);
    return set_last_error(FA_ERR_INVALID, msg);
  }
  if (r.rotary_dim > 0 && (!r.turns || (reinterpret_cast<uintptr_t>(r.turns) & 7u))) {
    snprintf(msg, sizeof(msg), "%s: turns is NULL or not 8-byte aligned", who);
    return set_last_error(FA_ERR_INVALID, msg);
  }
  return FA_OK;
}

template <typename T>
cudaError_t launch_rotary(RotaryArgs& a, bool vec, cudaStream_t stream) {
  const int heads = a.H + a.Hkv;
  a.units = vec ? a.D / 16 : (a.D + 1) / 2;
  const int64_t n = (int64_t)a.B * a.T * a.units;
  a.heads_per_thread = heads_per_thread(n, heads);
  const unsigned x = (unsigned)((n + 255) / 256);
  const int hpt = a.heads_per_thread;
  a.q_chunks = (a.H + hpt - 1) / hpt;
  if (vec) rotary_kernel<T><<<dim3(x, a.q_chunks + (a.Hkv + hpt - 1) / hpt), 256, 0, stream>>>(a);
  else rotary_pair_kernel<T><<<dim3(x, (heads + hpt - 1) / hpt), 256, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, bool E4M3>
cudaError_t launch_append(AppendArgs& a, cudaStream_t stream) {
  const int64_t teams = (int64_t)a.B * a.pages_per_seq * a.Hkv * 2;
  const int rows = std::min(a.T, a.ps);
  const bool warp = rows * a.units <= 64;
  // A team is a warp when the rows that one page can take fit its registers, else a block.  Two passes for
  // 8-bit pages whose rows 256 threads then hold: with 64 registers a thread, and one of q's heads in work,
  // a third more threads share an SM (pages of 64 rows of 128: 59 us, with four passes and two heads 66; of
  // 128 rows, which would take 512 threads: 66 against 59).  bf16 pages, which need no second pass over the
  // values: 57 with two, 54 with four.
  const int passes = warp || (E4M3 && a.ps * a.units <= 512) ? 2 : 4;
  const int nt = warp ? 128 : std::max(64, a.ps * a.units / passes);
  a.kv_blocks = (int)(warp ? (teams + 3) / 4 : teams);
  int qb = 0;
  if (a.H > 0) {
    const int64_t n = (int64_t)a.B * a.T * a.units;
    a.heads_per_thread = heads_per_thread(n, a.H);
    a.q_blocks = (int)((n + nt - 1) / nt);
    qb = a.q_blocks * ((a.H + a.heads_per_thread - 1) / a.heads_per_thread);
  }
  const unsigned grid = (unsigned)(a.kv_blocks + qb);
  if (warp) {
    append_kernel<T, E4M3, true, 2, 128><<<grid, nt, 0, stream>>>(a);
    return cudaGetLastError();
  }
  const auto kernel = passes == 2 ? append_kernel<T, E4M3, false, E4M3 ? 2 : 4, 256>  // (8-bit only)
                      : nt <= 256 ? append_kernel<T, E4M3, false, 4, 256>
                                  : append_kernel<T, E4M3, false, 4, 512>;
  const size_t smem = E4M3 && a.r.rotary_dim ? (size_t)nt * passes * 4 * sizeof(float4) : 0;  // up to 128 KB
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  kernel<<<grid, nt, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace

int check_paged_cache(const FaPagedCache& c, int B, const char* who) {
  char msg[224];
  auto fail = [&](int code, const char* what) {
    snprintf(msg, sizeof(msg), "%s: %s", who, what);
    return set_last_error(code, msg);
  };
  if (c.dtype != FA_DTYPE_BF16 && c.dtype != FA_DTYPE_E4M3) return fail(FA_ERR_INVALID, "the cache must be bf16 or e4m3");
  if (c.num_pages <= 0 || c.H_kv <= 0 || c.table_cols <= 0 || B <= 0)
    return fail(FA_ERR_INVALID, "non-positive shape (num_pages, H_kv, table_cols or B)");
  if (c.page_size != 16 && c.page_size != 32 && c.page_size != 64 && c.page_size != 128)
    return fail(FA_ERR_UNSUPPORTED, "page_size must be 16, 32, 64 or 128");
  if (c.D != 64 && c.D != 128 && c.D != 256) return fail(FA_ERR_UNSUPPORTED, "head dim must be 64, 128 or 256");
  if ((int64_t)c.table_cols * c.page_size > (1 << 30)) return fail(FA_ERR_UNSUPPORTED, "more than 2^30 positions a sequence");
  if (!c.k.ptr || !c.v.ptr || !c.block_table) return fail(FA_ERR_INVALID, "NULL cache or block table");
  if (c.table_stride < 0) return fail(FA_ERR_INVALID, "negative block-table stride");
  const int es = c.dtype == FA_DTYPE_E4M3 ? 1 : 2;
  for (const FaTensor* t : {&c.k, &c.v}) {
    if (t->stride_b < 0 || t->stride_h < 0 || t->stride_t < c.D) return fail(FA_ERR_INVALID, "bad cache strides");
    if (!vec_ok(*t, es)) return fail(FA_ERR_INVALID, "cache base and strides must be multiples of 16 bytes");
  }
  if (c.dtype == FA_DTYPE_E4M3 && (!c.k_scale || !c.v_scale)) return fail(FA_ERR_INVALID, "an e4m3 cache needs k_scale and v_scale");
  return FA_OK;
}

}  // namespace fa

using namespace fa;

extern "C" {

int fa_rotary(const FaRotaryParams* p, fa_stream_t stream) {
  char msg[192];
  if (!p) return set_last_error(FA_ERR_INVALID, "fa_rotary: params is NULL");
  if (p->dtype != FA_DTYPE_BF16 && p->dtype != FA_DTYPE_F32) return set_last_error(FA_ERR_INVALID, "fa_rotary: unknown dtype");
  if (p->B <= 0 || p->H < 0 || p->H_kv < 0 || p->H + p->H_kv <= 0 || p->T <= 0 || p->D <= 0) {
    snprintf(msg, sizeof(msg), "fa_rotary: non-positive shape B=%d H=%d H_kv=%d T=%d D=%d", p->B, p->H, p->H_kv, p->T, p->D);
    return set_last_error(FA_ERR_INVALID, msg);
  }
  int rc = check_spec(p->rotary, p->D, "fa_rotary");
  if (rc) return rc;
  if ((int64_t)p->B * p->T * ((p->D + 1) / 2) >= (int64_t)1 << 31)
    return set_last_error(FA_ERR_UNSUPPORTED, "fa_rotary: B * T * D / 2 must stay below 2^31");
  if (!p->positions && (int64_t)p->pos_offset + p->T > (int64_t)1 << 31)
    return set_last_error(FA_ERR_INVALID, "fa_rotary: positions from pos_offset on do not fit 32 bits");
  if ((int64_t)p->H + p->H_kv > 65535) return set_last_error(FA_ERR_UNSUPPORTED, "fa_rotary: more than 65535 heads");
  const int es = p->dtype == FA_DTYPE_F32 ? 4 : 2;
  bool vec = p->D % 16 == 0 && p->rotary.rotary_dim % 16 == 0;
  for (int i = 0; i < 2; ++i) {
    const FaTensor &x = i ? p->k : p->q, &y = i ? p->k_out : p->q_out;
    if ((i ? p->H_kv : p->H) == 0) continue;
    if (!x.ptr || !y.ptr) return set_last_error(FA_ERR_INVALID, "fa_rotary: NULL tensor");
    vec = vec && vec_ok(x, es) && vec_ok(y, es);
  }
  RotaryArgs a;
  a.B = p->B; a.H = p->H; a.Hkv = p->H_kv; a.T = p->T; a.D = p->D;
  a.q = p->q; a.k = p->k; a.q_out = p->q_out; a.k_out = p->k_out;
  a.positions = p->positions; a.pos_stride_b = p->pos_stride_b; a.pos_offset = p->pos_offset;
  a.sign = p->inverse ? -1.f : 1.f;
  a.r = p->rotary;
  cudaError_t e = p->dtype == FA_DTYPE_F32 ? launch_rotary<float>(a, vec, (cudaStream_t)stream)
                                           : launch_rotary<__nv_bfloat16>(a, vec, (cudaStream_t)stream);
  if (e != cudaSuccess) {
    snprintf(msg, sizeof(msg), "fa_rotary: %s", cudaGetErrorString(e));
    return set_last_error(FA_ERR_CUDA, msg);
  }
  return FA_OK;
}

int fa_paged_append(const FaPagedAppendParams* p, fa_stream_t stream) {
  char msg[192];
  if (!p) return set_last_error(FA_ERR_INVALID, "fa_paged_append: params is NULL");
  if (p->dtype != FA_DTYPE_BF16 && p->dtype != FA_DTYPE_F32)
    return set_last_error(FA_ERR_INVALID, "fa_paged_append: unknown dtype");
  int rc = check_paged_cache(p->cache, p->B, "fa_paged_append");
  if (rc) return rc;
  if (p->T <= 0 || p->H < 0) return set_last_error(FA_ERR_INVALID, "fa_paged_append: non-positive T or negative H");
  if ((rc = check_spec(p->rotary, p->cache.D, "fa_paged_append"))) return rc;
  if (p->rotary.rotary_dim % 16) return set_last_error(FA_ERR_UNSUPPORTED, "fa_paged_append: rotary_dim must be a multiple of 16");
  if (!p->k.ptr || !p->v.ptr || !p->kv_lens || (p->H > 0 && (!p->q.ptr || !p->q_out.ptr)))
    return set_last_error(FA_ERR_INVALID, "fa_paged_append: NULL tensor");
  const FaPagedCache& c = p->cache;
  const int es = p->dtype == FA_DTYPE_F32 ? 4 : 2;
  AppendArgs a;
  a.B = p->B; a.H = p->H; a.T = p->T; a.Hkv = c.H_kv; a.D = c.D; a.ps = c.page_size; a.num_pages = c.num_pages;
  a.cols = c.table_cols; a.table_stride = c.table_stride; a.table = c.block_table;
  a.units = c.D / 16;
  // pages that T new tokens can touch, wherever in a page they start
  a.pages_per_seq = (int)std::min<int64_t>(c.table_cols, ((int64_t)p->T + c.page_size - 2) / c.page_size + 1);
  a.heads_per_thread = 1; a.q_blocks = 1;
  a.q = p->q; a.k = p->k; a.v = p->v; a.q_out = p->q_out; a.kc = c.k; a.vc = c.v;
  a.k_scale = c.k_scale; a.v_scale = c.v_scale;
  a.kv_lens = p->kv_lens; a.new_lens = p->new_lens;
  a.r = p->rotary; a.status = p->status;
  a.vec = vec_ok(p->k, es) && vec_ok(p->v, es) && (p->H == 0 || (vec_ok(p->q, es) && vec_ok(p->q_out, es)));
  if ((int64_t)p->B * a.pages_per_seq * c.H_kv * 2 >= (int64_t)1 << 30 ||
      (int64_t)p->B * p->T * a.units * std::max(1, p->H) >= (int64_t)1 << 31)
    return set_last_error(FA_ERR_UNSUPPORTED, "fa_paged_append: too many new tokens for one call");
  cudaError_t e;
  const cudaStream_t st = (cudaStream_t)stream;
  if (c.dtype == FA_DTYPE_E4M3)
    e = es == 4 ? launch_append<float, true>(a, st) : launch_append<__nv_bfloat16, true>(a, st);
  else
    e = es == 4 ? launch_append<float, false>(a, st) : launch_append<__nv_bfloat16, false>(a, st);
  if (e != cudaSuccess) {
    snprintf(msg, sizeof(msg), "fa_paged_append: %s", cudaGetErrorString(e));
    return set_last_error(FA_ERR_CUDA, msg);
  }
  return FA_OK;
}

}  // extern "C"
