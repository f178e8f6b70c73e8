// Attention of query rows against a paged K/V cache (fa_paged_attn), bf16 or 8-bit (e4m3).
//
// Per query row: x_j = score(scale * q . k_j), o = sum_j softmax(x)_j v_j, with k_j = ks * code and
// v_j = vs * code where ks, vs belong to the page and K/V head of position j.  A decode step reads
// every cached byte once and does a few multiply-adds with each, so HBM bounds it; a prompt
// chunk is bound by the tensor cores and the exponentials.
//
// Orientation.  The 128 cached positions of a tile are the MMA's M, the query rows its N:
//     S^T [128 positions x R] = K Q^T       A = K as stored (K-major), B = Q
//     O^T [D x R]            += V^T P^T     A = V as stored (M-major), B = P from shared memory
// so the exponentials are spent on real query rows only (R is 8 to 64 of them; with the rows as M
// they would be padded to 128), and each thread owns one position: its page's scales are two
// registers.
//
// 8-bit codes go to the tensor cores as they are (kind::f8f6f4): converting a tile in shared memory
// would cost as many instructions as everything else here.  The other operand is split into two e4m3
// parts, z = hi + lo, that meet in the fp32 accumulator: both parts' MMAs add to the same columns
// (R >= 16), or for R = 8 the parts lie side by side in the MMA's smallest N of 16 and are added
// when read.  q is scaled by a power of two per row so that its largest magnitude lies in [128, 256):
// a bf16 has 8 significant bits, each part 4, so the split is exact down to 2^-17 of the row's largest
// element.  Probabilities lie in [0, 431], the largest of a tile that moved the reference at 32: hi
// is P cut to 4 bits, lo the rest rounded to 4, off by 2^-8 relative (as a bf16 P is) or by 2^-15 of
// the largest below that.
//
// Scales.  ks multiplies the thread's logits.  vs goes into the exponent: with z = x + log2 vs and
// a reference m per row, P = 2^(z - m + 7) weighs the codes, and the softmax sum adds P / vs;
// o = sum P code / sum (P / vs).  So a row whose weight sits on pages of small values keeps its
// precision.  A reference moves up when a tile exceeds it by more than 1.75: one barrier vote per
// tile.  A unit's tiles are taken from its end to its start: under ALiBi, and mostly without it, the
// largest logits come first and the references hardly move.
// An 8-bit reference moves down again, too, by up to 20 below its highest: the smallest step of the
// parts is 2^-9, and a tile far below the reference would keep its place in the sum and lose it in O (a key
// 11 nats above a rest of 32768 positions: o off by 5 to 10 %, now 0.2 at most).  When a row's largest P was below
// 1/2 in two tiles, the third one's becomes 32, and O and the sum are scaled up.  (After one such tile there
// would be twice as many moves where neighbouring tiles differ in size.  For the prompt chunk below, whose
// pages' scales differ by up to 8, references that move down cost 27 us of 262, for decode 1 of 75.)
//
// Work.  The tiles of all (sequence, row group, K/V head) units, in that order, are cut into equal
// contiguous ranges, one per CTA (one CTA per SM): ragged batches balance themselves, and nothing
// about the lengths is needed on the host.  A unit inside one CTA is written to o directly; one
// that crosses CTAs leaves at most one partial (o, lse) at each end of a CTA's range in the
// workspace; after a grid barrier (the launch is cooperative) the CTA that holds a unit's first part
// joins its parts in CTA order.  A second kernel for that took 5-6 us more on the device and 6 us
// on the host; counters or flags in the workspace would have to be zero before the call.
//
// Warps: softmax groups of four (thread = position of a tile; at the end = element of D), then one or
// two that produce K and V (lane = page of a tile), one that issues S, one that issues P V, and one that builds
// the next unit's Q operand and row constants.  A group works on up to 16 rows.  Up to 32 rows there
// are two sets of groups that take the tiles in turn, each with its own O, references and sums: a
// tile's chain (wait, TMEM read, vote, exponentials, store, fence) takes longer than its bytes take to
// arrive, so two tiles have to be in work at once.  The set that took a unit's last tile joins and
// writes its two O, while the other one, having posted its sums, is already in the next unit (O and
// sums are double-buffered for that).  64 rows leave threads for one set only.
//
// Measured on the device (8-bit pages, H 32, H_kv 8, D 128, ragged lengths): 64 users of up to 4096
// positions, one token each: 75 us, 5.3 TB/s, 0.82 of the measured copy rate; eight of up to 32768: 74 us,
// 5.4 TB/s; one of 1000: 10 us, the launch, one tile's chain and the join.  Chunks of 512 tokens of four
// users on up to 4096 positions: 265 us, bound by the chain of one set of softmax groups at 64 rows.
// bf16, H 16, D 64, window 1024, ALiBi, 32 users: 46 us.
#include <cooperative_groups.h>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdio>

#include "fa_common.cuh"
#include "fa_internal.h"
#include "fa_ptx.cuh"
#include "flexattn.h"

namespace fa {
namespace {

constexpr int kTile = 128;         // cached positions of a tile: the MMA's M
constexpr int kMaxSlots = 24;      // K or V tiles in the shared-memory ring
constexpr int kScaleRing = 16;     // tiles whose scales may be live at once (> kMaxSlots / 2 + 1)
// A reference moves when exceeded by more than slack (log2 units), to head above the tile's largest z;
// P = 2^(z - reference + lift).  8-bit: P in units of 2^-8, so that fp16's exponents line up with
// e4m3's (split_e4m3x4), at most 2^(7 + 1.75) = 431, below e4m3's 448; the head spares most moves
// (each costs about half a tile's time) for two bits at the small end.  bf16 holds 2^60 as well as 1.
__host__ __device__ constexpr float slack_of(int ES) { return ES == 1 ? 1.75f : 60.f; }
__host__ __device__ constexpr float head_of(int ES) { return ES == 1 ? 2.f : 0.f; }
__host__ __device__ constexpr float lift_of(int ES) { return ES == 1 ? 7.f - 8.f : 0.f; }
// Value scales.  The append's least one, 2^-100, and less count as zero: the page's codes are cleared, and
// since its place in the exponent is free then, it is one that keeps sums in range and does not push the
// reference up.  In tiles with such a page, or one of a scale far from 1, P / vs is not formed from P, which
// may have underflowed (next to a page of 2^30, P of one of 2^-90 is 2^-120 at the same logit), but from the
// logit.  (A choice in the common loop instead of a loop before it took 247 instead of 235 us for the prompt
// chunk below.)
constexpr float kNoScale = 0x1p-100f, kScaleless = 0x1p-80f, kFar2 = 0x1p40f;
constexpr uint32_t kZeros = 1u, kSigns = 0x80808080u, kNaNs = 0x7f7f7f7fu;  // codes that become 0, change sign, or become NaN
constexpr int kCleared = 1, kFar = 2;  // a tile with a hidden page or one whose scale is not above 2^-100 and
                                       // finite (negative ones are for the codes' signs); with one far from 1
constexpr float kUnset = -1e30f;   // reference of a row that has seen nothing yet
constexpr float kDrop = 20.f;      // 8-bit: how far a reference goes below the highest one it had

struct PagedArgs {
  int B, H, Hkv, Tq, G, M;         // M = G * Tq query rows per sequence and K/V head
  int ps_log, cols, num_pages, groups; // groups of R query rows per (sequence, K/V head)
  int entries;                     // B * groups
  int slots;                       // ring depth
  int q_vec;
  int64_t table_stride;
  FaTensor q, o;
  float* lse;
  const int32_t *kv_lens, *q_lens, *table;
  const float *k_scale, *v_scale;
  float scale;
  FaMaskSpec mask;
  FaScoreSpec score;
  float* part_o;    // [2 * CTAs][R][D]
  float* part_lse;  // [2 * CTAs][R]
  int joins;        // a unit may cross CTAs: the launch is cooperative
  int* status;
};

template <int D, int ES, int R>
struct Shape {
  static constexpr bool SIDE = ES == 1 && R == 8;   // hi and lo parts side by side in N
  static constexpr bool TURNS = R <= 32;            // two sets of softmax groups take the tiles in turn
  static constexpr int H = R <= 16 ? 1 : R / 16;    // groups in a set, 16 rows (or all) each
  static constexpr int NG = TURNS ? 2 * H : H;
  static constexpr int NSM = 128 * NG;              // softmax threads
  static constexpr int LOADERS = R == 8 ? 2 : 1;    // warps that produce: K and V, or both
  static constexpr int NT = NSM + 32 * (LOADERS + 3);
  static constexpr int N = SIDE ? 16 : R;           // columns of S and O
  static constexpr int C = R < 16 ? R : 16;         // rows per softmax thread
  static constexpr int PARTS = ES == 1 && !SIDE ? 2 : 1;  // operands of Q and P (hi, lo)
  static constexpr int ROWB = D * ES;               // bytes of one cached position
  static constexpr int SW = ROWB < 128 ? 64 : 128;  // swizzle span
  static constexpr int PANEL = kTile * SW;
  static constexpr int SLOT = kTile * ROWB;
  static constexpr int QPANEL = N * SW;
  static constexpr int QPART = N * ROWB, QBUF = PARTS * QPART;
  static constexpr int PPART = N * kTile * ES, PBUF = PARTS * PPART;
  static constexpr int NO = D <= 128 ? 1 : D / 128; // blocks of 128 elements of O
  static constexpr int ON = NO * N;                 // TMEM columns of one O
  static constexpr uint32_t TM_O = 2 * N;           // TMEM: two S buffers, then one O, or one per group and unit parity
  static constexpr int USED = 2 * N + (TURNS ? 4 : 1) * ON;
  static constexpr uint32_t TM_COLS = USED <= 32 ? 32 : USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static_assert(USED <= 512 && N % 16 == 0 && N <= 256 && (ES == 1 || R >= 16), "operand shape");
};

// One CTA's part of a unit, as the walk finds it.
struct Seg {
  int hk, t0, nt;      // K/V head, first tile taken (they go down from there), tiles
  int first, last;     // holds the unit's first / last tile in that order
  int rows;            // query rows of the group
  int lo, hi, in_lo, in_hi;  // of its entry
  int entry, entry_nt;
};

// Description and row constants of one unit (double-buffered with Q).
template <int R> struct RowConst {
  Seg sg;
  float xs[R];      // logit = dot * (ks * xs): scale, the row's power of two, and log2(e) unless softcapped
  float slope[R];   // ALiBi slope in the same domain
  int lo[R], hi[R]; // positions the row may see; hi < lo: none
  int qpos[R];
  int64_t qoff[R];  // element offset of the row in q, -1: nothing to read
  int64_t orow[R];  // the same in o, -1: no such row
  int64_t lrow[R];  // index of the row in lse
};
// Running state of one softmax group: its rows, or its share of the tiles.
struct RowState {
  float m[16], bias[16];  // reference; lift - reference
  float move[16];         // factor of the last move
  float high[16];         // the highest reference so far (8-bit)
  uint4 seen[2];          // rows with a probability of 1/2 or more in the last two tiles (row_bit), by warp; in turn
  uint32_t watch;         // rows whose reference may go down
  int far;                // a value scale far from 1 was met: none may, so that sums stay in range
  float4 red[16];         // a value of each warp
  float fin[2][16];       // factors of the O (of both groups) at the end; the first negative: no position seen
};
struct Posted {  // what a group knows of a unit when it leaves it
  float m[16];
  float4 sum[16];  // a part of each warp
};
// What one (sequence, row group) has to visit.
struct Entry {
  int b, rg, len, ql;
  int lo, hi;        // positions that some row of the group may see
  int in_lo, in_hi;  // positions that every valid row of the group may see
  int t0, nt;        // tiles
};

template <int R>
__device__ __forceinline__ Entry entry_of(const PagedArgs& a, int e) {
  Entry x;
  x.b = a.groups == 1 ? e : e / a.groups;
  x.rg = e - x.b * a.groups;
  const int cap = a.cols << a.ps_log;
  const int len = __ldg(a.kv_lens + x.b), ql = a.q_lens ? __ldg(a.q_lens + x.b) : a.Tq;
  x.len = min(max(len, 0), cap);
  x.ql = min(max(ql, 0), a.Tq);
  int i0 = 0, i1 = a.Tq - 1;  // tokens of the group's rows
  if (a.groups > 1) {
    i0 = x.rg * R / a.G;
    i1 = (min(x.rg * R + R, a.M) - 1) / a.G;
  }
  i1 = min(i1, x.ql - 1);
  const int p0 = x.len - x.ql + i0, p1 = x.len - x.ql + i1;  // positions of the group's rows
  x.lo = 0;
  x.hi = x.len - 1;
  x.in_lo = 0;
  x.in_hi = x.len - 1;
  if (a.mask.flags & FA_MASK_CAUSAL) {
    x.hi = min(x.hi, p1);
    x.in_hi = min(x.in_hi, p0);
  }
  if (a.mask.flags & FA_MASK_WINDOW) {
    if (a.mask.window_left >= 0) {
      x.lo = max(x.lo, p0 - a.mask.window_left);
      x.in_lo = max(x.in_lo, p1 - a.mask.window_left);
    }
    if (a.mask.window_right >= 0) {
      x.hi = min(x.hi, (int)min((int64_t)p1 + a.mask.window_right, (int64_t)x.len));
      x.in_hi = min(x.in_hi, (int)min((int64_t)p0 + a.mask.window_right, (int64_t)x.len));
    }
  }
  x.t0 = x.lo / kTile;
  x.nt = (i1 < i0 || x.hi < x.lo) ? 0 : x.hi / kTile - x.t0 + 1;
  return x;
}

// One CTA's range of tiles, unit by unit, is walked by the producer (each lane for itself) and by the
// warp that builds Q, which describes each unit's part to the others.
struct Start {  // where a CTA's range begins
  Entry e;
  int idx, hk, off;
};
template <int R>
struct Walker {
  Entry e;
  int idx, hk, off, left;
  __device__ __forceinline__ void begin(const Start& s, int tiles) {
    left = tiles;
    e.nt = 0;
    if (tiles > 0) {
      e = s.e;
      idx = s.idx;
      hk = s.hk;
      off = s.off;
    }
  }
  // Moves tiles beyond a unit's end on into the next head, or the next entry that has tiles.
  __device__ __forceinline__ void settle(const PagedArgs& a) {
    while (off >= e.nt) {
      off -= e.nt;
      if (e.nt > 0 && ++hk < a.Hkv) continue;
      hk = 0;
      e = entry_of<R>(a, ++idx);
    }
  }
  __device__ __forceinline__ bool next(const PagedArgs& a, Seg* s) {
    if (left <= 0) return false;
    settle(a);
    s->hk = hk;
    s->t0 = e.t0 + e.nt - 1 - off;
    s->nt = min(e.nt - off, left);
    s->first = off == 0;
    off += s->nt;
    s->last = off == e.nt;
    left -= s->nt;
    s->rows = a.M - e.rg * R;
    s->lo = e.lo;
    s->hi = e.hi;
    s->in_lo = e.in_lo;
    s->in_hi = e.in_hi;
    s->entry = idx;
    s->entry_nt = e.nt;
    return true;
  }
};

template <int R> struct Smem {
  RowConst<R> rc[2];
  RowState rs[R <= 16 ? 2 : 4];
  Posted post[2][R <= 16 ? 2 : 4];  // by unit parity and group
  float2 scales[kScaleRing][8];  // (ks, |vs|) of a tile's pages; ks = -inf hides the page; vs may be kScaleless
  uint32_t turned[kScaleRing][8];  // what becomes of a page's V codes: 0 (they stay), kZeros, kSigns, kNaNs
  int odd[kScaleRing];           // kCleared, kFar: what the tile's pages ask for beside the common path
  // A slot's loads of K and of V complete on a barrier each: where the ring has an odd number of slots, a slot
  // holds K and V in turn, and a reader that waits for K by the parity of a common barrier would pass while
  // the slot's V before it has not landed (its own readers may be behind).
  uint64_t full_k[kMaxSlots], full_v[kMaxSlots], empty[kMaxSlots], s_full[2], p_full[2], o_full[2], q_full[2], q_empty[2], posted[2], done[2], fin_bar[2];
  int scan[24];
  Start start;
  // the unit whose first part this CTA holds: how many parts it has (0: no such unit), the first one's
  // slot (the others' is 2 k of the CTAs k that follow), its entry and K/V head
  int join_parts, join_slot, join_entry, join_hk;
  int empties, empty_entry[64];  // entries without a tile of which this CTA writes heads cta - entry, + CTAs, ...
  uint32_t tmem;
  int abort_flag, never;
};

template <int D, int ES, int R>
size_t paged_smem_bytes(int slots) {
  using S = Shape<D, ES, R>;
  return 1024 + (size_t)slots * S::SLOT + 2 * S::QBUF + 2 * S::PBUF + sizeof(Smem<R>);
}

// Bounded wait for a barrier's phase; false when the CTA gave up or after kSpins polls: between 50 ms
// (every poll answers at once) and some seconds (the hardware lets polls sleep), where the longest
// legitimate wait of this kind is that of a tile or a unit's Q operand, microseconds.  Only the warp
// that builds Q waits for whole units, with mbar_wait's bound on time.  No clock here: two dozen waits
// in line fill the instruction cache, and the shorter one took 10 % off the windowed case.
// A warp's lanes may leave the polls one by one, and what follows a wait is for whole warps (tcgen05.ld and
// bar.sync are .aligned): so they meet again here.  Called by whole warps only.
constexpr uint32_t kSpins = 1u << 20;
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  bool there = false;
#pragma unroll 1
  for (uint32_t n = 0; n < kSpins; ++n) {
    there = mbar_try_wait(bar, parity);
    if (there || *abort_flag) break;
  }
  __syncwarp();
  return there;
}
__device__ __forceinline__ bool wait_for_w(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  const int ok = wait_for(bar, parity, abort_flag) ? 1 : 0;
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// A named barrier for whole warps, whose lanes may come from a branch.
__device__ __forceinline__ void bar_sync_w(int id, int nthreads) {
  __syncwarp();
  named_bar_sync(id, nthreads);
}
__device__ __forceinline__ bool vote_or(int id, int nthreads, bool pred) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(nthreads), "r"((uint32_t)pred)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint32_t e4m3x2(__half2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(*reinterpret_cast<const uint32_t*>(&v)));
  return r;
}
__device__ __forceinline__ __half2 e4m3x2_value(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return *reinterpret_cast<const __half2*>(&h);
}
// Two values of magnitude up to 448 as hi + lo: packed hi parts, lo parts through *lo2.  Between the
// two parts the value passes through fp16: 11 bits, finer than both.
__device__ __forceinline__ uint32_t split_e4m3x2(float a, float b, uint32_t* lo2) {
  const __half2 v = __floats2half2_rn(a, b);
  const uint32_t h = e4m3x2(v);
  *lo2 = e4m3x2(__hsub2(v, e4m3x2_value(h)));
  return h;
}
// The same for four values >= 0 in units of 2^-8 (so at most 1.75), with integer operations: an fp16
// in these units is the e4m3 code shifted left by 7 bits, down to the subnormal ones, so cutting an
// fp16 to its upper 9 bits is a truncation to e4m3.  The conversion instructions (three for two
// values) run at a fraction of the rate and bounded the kernel at 64 rows.  NaN stays NaN.
__device__ __forceinline__ uint32_t split_e4m3x4(const float (&p)[4], uint32_t* lo4) {
  const __half2 a = __floats2half2_rn(p[0], p[2]), b = __floats2half2_rn(p[1], p[3]);
  uint32_t ha = *reinterpret_cast<const uint32_t*>(&a) & 0x7f807f80u, hb = *reinterpret_cast<const uint32_t*>(&b) & 0x7f807f80u;
  const __half2 ra = __hsub2(a, *reinterpret_cast<const __half2*>(&ha)), rb = __hsub2(b, *reinterpret_cast<const __half2*>(&hb));
  const uint32_t la = (*reinterpret_cast<const uint32_t*>(&ra) + 0x00400040u) & 0x7f807f80u,
                 lb = (*reinterpret_cast<const uint32_t*>(&rb) + 0x00400040u) & 0x7f807f80u;
  *lo4 = (la >> 7) | (lb << 1);
  return (ha >> 7) | (hb << 1);
}

// Row n's bit in a mask of 16 rows, as split_e4m3x4's codes give it: byte n % 4 of word n / 4, whose
// upper bits lie side by side.
__host__ __device__ constexpr uint32_t row_bit(int n) { return 0x80u << (8 * (n & 3)) >> (n >> 2); }

// Byte offset of 16-byte chunk c of row r in a panel of rows of SW bytes, swizzled over SW.
template <int SW>
__device__ __forceinline__ uint32_t panel_off(int r, int c) {
  return (uint32_t)(r * SW + ((SW == 128 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3))) << 4));
}

// Sums of C values over a warp: lane l ends with the sum of column l * C / 32 (lanes of the same
// column hold the same).  Each step exchanges the half of the columns that the partner keeps.
template <int C>
__device__ __forceinline__ float warp_col_sums(float (&v)[C], int lane) {
  int o = 16;
#pragma unroll
  for (int h = C / 2; h >= 1; h /= 2, o /= 2) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int k = 0; k < h; ++k) {
      const float give = up ? v[k] : v[k + h], keep = up ? v[k + h] : v[k];
      v[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
  float r = v[0];
#pragma unroll
  for (; o; o /= 2) r += __shfl_xor_sync(0xffffffffu, r, o);
  return r;
}

// Row constants of a unit's row group and K/V head but for xs, and where its rows of q are (in qoff):
// one thread a row.
template <int R>
__device__ __forceinline__ void build_rows(const PagedArgs& a, const Entry& e, int hk, RowConst<R>& rc, int t, int nt) {
  const float dom = (a.score.flags & FA_SCORE_SOFTCAP) ? 1.f : kLog2e;
  for (int n = t; n < R; n += nt) {
    const int m = e.rg * R + n, i = m / a.G, h = hk * a.G + (m - i * a.G);
    const bool real = m < a.M, live = real && i < e.ql;
    const int qpos = e.len - e.ql + i;
    int lo = 0, hi = e.len - 1;
    if (a.mask.flags & FA_MASK_CAUSAL) hi = min(hi, qpos);
    if (a.mask.flags & FA_MASK_WINDOW) {
      if (a.mask.window_left >= 0) lo = max(lo, qpos - a.mask.window_left);
      if (a.mask.window_right >= 0) hi = (int)min((int64_t)hi, (int64_t)qpos + a.mask.window_right);
    }
    rc.slope[n] = live && (a.score.flags & FA_SCORE_ALIBI) ? __ldg(a.score.alibi_slopes + h) * dom : 0.f;
    rc.lo[n] = live ? lo : 1;
    rc.hi[n] = live ? hi : 0;
    rc.qpos[n] = qpos;
    rc.qoff[n] = live ? (int64_t)e.b * a.q.stride_b + (int64_t)h * a.q.stride_h + (int64_t)i * a.q.stride_t : -1;
    rc.orow[n] = real ? (int64_t)e.b * a.o.stride_b + (int64_t)h * a.o.stride_h + (int64_t)i * a.o.stride_t : -1;
    rc.lrow[n] = ((int64_t)e.b * a.H + h) * a.Tq + i;
  }
}

// The Q operand of the rows that build_rows described, and their xs, by NT threads; rows that do not
// exist become zeros.
template <int D, int ES, int R, int NT>
__device__ __forceinline__ void build_q(const PagedArgs& a, unsigned char* q, RowConst<R>& rc, int t) {
  using S = Shape<D, ES, R>;
  constexpr int SW = S::SW;
  constexpr int TPR = D / 8;      // threads per row, 8 elements each
  constexpr int ROWS = NT / TPR;  // rows at once
  constexpr int PASSES = (R + ROWS - 1) / ROWS;
  constexpr int UN = PASSES < 4 ? PASSES : 4;  // rows in flight per thread
  const int d0 = (t % TPR) * 8;
  const float dom = (a.score.flags & FA_SCORE_SOFTCAP) ? 1.f : kLog2e;
#pragma unroll 1
  for (int p0 = 0; p0 < PASSES; p0 += UN) {
    uint4 raws[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int n = (p0 + u) * ROWS + t / TPR;
      raws[u] = make_uint4(0u, 0u, 0u, 0u);
      const int64_t off = n < R ? rc.qoff[n] : -1;
      if (off >= 0) {
        const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q.ptr) + off + d0;
        if (a.q_vec) {
          raws[u] = __ldg(reinterpret_cast<const uint4*>(qp));
        } else {
          raws[u].x = (uint32_t)qp[0] | ((uint32_t)qp[1] << 16);
          raws[u].y = (uint32_t)qp[2] | ((uint32_t)qp[3] << 16);
          raws[u].z = (uint32_t)qp[4] | ((uint32_t)qp[5] << 16);
          raws[u].w = (uint32_t)qp[6] | ((uint32_t)qp[7] << 16);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int n = (p0 + u) * ROWS + t / TPR;
      const uint4 raw = raws[u];
      float fix = 1.f;  // undoes the row's power of two
      if constexpr (ES == 2) {
        if (n < R) *reinterpret_cast<uint4*>(q + (d0 * 2 / SW) * S::QPANEL + panel_off<SW>(n, (d0 * 2 % SW) >> 4)) = raw;
      } else {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        // The largest magnitude: bf16 magnitudes compare as integers, NaN and infinity come out above all.
        uint32_t top = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) top = max(top, max((w[k] << 16) & 0x7fff0000u, w[k] & 0x7fff0000u));
#pragma unroll
        for (int o = TPR / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^sh brings it into [128, 256) (at most 2^100: tinier rows stay small)
        const bool finite = top < 0x7f800000u;
        const int sh = top > 0 && finite ? min(7 + 127 - (int)(top >> 23), 100) : 0;
        const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
        fix = finite ? __uint_as_float((uint32_t)(127 - sh) << 23) : __uint_as_float(0x7fc00000u);  // such a row is NaN
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          hi[k] = split_e4m3x2(__uint_as_float(w[k] << 16) * up, __uint_as_float(w[k] & 0xffff0000u) * up, &lo[k]);
        if (n < R) {
          unsigned char* at = q + (d0 / SW) * S::QPANEL + (d0 & 8);
          const int c = (d0 % SW) >> 4;
          *reinterpret_cast<uint2*>(at + panel_off<SW>(n, c)) = make_uint2(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
          *reinterpret_cast<uint2*>(at + (S::SIDE ? panel_off<SW>(R + n, c) : S::QPART + panel_off<SW>(n, c))) =
              make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
        }
      }
      if (d0 == 0 && n < R) rc.xs[n] = a.scale * fix * dom;
    }
  }
}

// o = 0 and lse = -inf for the rows of an entry without a tile, those heads that are this CTA's.
template <int D, int R>
__device__ __forceinline__ void empty_rows(const PagedArgs& a, int e, int cta, int warp, int warps, int lane) {
  const int b = a.groups == 1 ? e : e / a.groups, m0 = (e - b * a.groups) * R, rows = min(R, a.M - m0);
  int hk = cta - e % (int)gridDim.x;
  if (hk < 0) hk += gridDim.x;
  for (; hk < a.Hkv; hk += gridDim.x)
    for (int r = warp; r < rows; r += warps) {
      const int m = m0 + r, i = m / a.G, h = hk * a.G + m - i * a.G;
      uint16_t* o = reinterpret_cast<uint16_t*>(a.o.ptr) + (int64_t)b * a.o.stride_b + (int64_t)h * a.o.stride_h +
                    (int64_t)i * a.o.stride_t;
#pragma unroll
      for (int d = 0; d < D; d += 32) o[d + lane] = 0;
      if (lane == 0) a.lse[((int64_t)b * a.H + h) * a.Tq + i] = -INFINITY;
    }
}

// MODS: ALiBi or softcap (their code in the common loop costs the plain kernel a third of its time).
template <int D, int ES, int R, bool MODS>
__global__ void __launch_bounds__((Shape<D, ES, R>::NT), 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                      const PagedArgs a) {
  using S = Shape<D, ES, R>;
  constexpr int N = S::N, SW = S::SW, C = S::C, NG = S::NG, NSM = S::NSM, NT = S::NT;
  constexpr int W_LOAD = 4 * NG, W_S = W_LOAD + S::LOADERS, W_PV = W_S + 1, W_Q = W_S + 2;  // warps behind the softmax
  constexpr bool TURNS = S::TURNS;
  constexpr uint32_t LAYOUT = SW == 128 ? SMEM_SWIZZLE_128B : SMEM_SWIZZLE_64B;
  constexpr int KPOS = 32 / ES;  // positions per PV MMA
  constexpr uint32_t IDESC_S = ES == 1 ? make_idesc_e4m3(128, N, 0, 0) : make_idesc_bf16(128, N, 0, 0);
  constexpr uint32_t IDESC_PV = ES == 1 ? make_idesc_e4m3(128, N, 1, 1) : make_idesc_bf16(128, N, 1, 1);

  extern __shared__ unsigned char dsm_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dsm_raw) + 1023) & ~uintptr_t(1023));
  const int NS = a.slots, turn = NS & 1 ? NS : NS / 2;  // tiles until K (or V) comes to the same slot again
  unsigned char* sQ = base + (size_t)NS * S::SLOT;
  unsigned char* sP = sQ + 2 * S::QBUF;
  Smem<R>& sm = *reinterpret_cast<Smem<R>*>(sP + 2 * S::PBUF);
  volatile int* abort_flag = &sm.abort_flag;
  volatile int* never = &sm.never;  // stays 0: waits on it end by their polls only

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;

  // ---------------------------------------------------------------- setup: barriers, TMEM, range
  if (tid == NT - 1) {  // (the first warps have entries to count)
    for (int i = 0; i < NS; ++i) {
      mbar_init(sm.full_k + i, 1);
      mbar_init(sm.full_v + i, 1);
      mbar_init(sm.empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sm.s_full + i, 1);
      mbar_init(sm.p_full + i, 4 * S::H);
      mbar_init(sm.o_full + i, 1);
      mbar_init(sm.q_full + i, 1);
      mbar_init(sm.q_empty + i, 2 + 4 * NG);  // the S issuer's commit, the P V issuer and the softmax warps
      mbar_init(sm.posted + i, 4 * S::H);  // a set's warps: the one that does not write the unit
      mbar_init(sm.done + i, 4 * S::H);    // the other one's: the unit is written
      mbar_init(sm.fin_bar + i, 1);
    }
    sm.abort_flag = 0;
    sm.never = 0;
    sm.join_parts = 0;
    sm.empties = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == W_S) {
    tmem_alloc(&sm.tmem, S::TM_COLS);
    tmem_relinquish();
  }
  int my_tiles, my_start, per;
  {
    // Exclusive prefix of the entries' tiles over the threads, each with a run of entries.
    const int run = (a.entries + NT - 1) / NT, e0 = min(tid * run, a.entries), e1 = min(e0 + run, a.entries);
    int mine = 0;
    Entry x;
    for (int e = e0; e < e1; ++e) {
      x = entry_of<R>(a, e);
      mine += x.nt * a.Hkv;
      if (x.rg == 0 && cta == 0) {
        const int n = __ldg(a.kv_lens + x.b), t = a.q_lens ? __ldg(a.q_lens + x.b) : 0;
        if (n < 0 || n > a.cols << a.ps_log || t < 0 || t > a.Tq) report_status(a.status, FA_ERR_INVALID);
      }
    }
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) sm.scan[warp] = inc;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      const int v = sm.scan[w];
      if (w < warp) before += v;
      total += v;
    }
    per = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int start = (int)min((int64_t)cta * per, (int64_t)total);
    my_start = start;
    my_tiles = min(per, total - start);
    for (int e = e0; e < e1; ++e) {
      if (run > 1) x = entry_of<R>(a, e);
      if (x.nt) continue;
      int hk = cta - e % (int)gridDim.x;  // some of its heads' rows are this CTA's to write
      if (hk < 0) hk += gridDim.x;
      if (hk < a.Hkv) {
        const int k = atomicAdd(&sm.empties, 1);
        if (k < 64) sm.empty_entry[k] = e;
      }
    }
    int at = before + inc - mine;
    if (start < total && at <= start && start < at + mine) {  // the range begins in one of this thread's entries
      for (int e = e0; e < e1; ++e) {
        if (run > 1) x = entry_of<R>(a, e);
        const int n = x.nt * a.Hkv;
        if (start < at + n) {
          sm.start.e = x;
          sm.start.idx = e;
          sm.start.hk = (start - at) / x.nt;
          sm.start.off = start - at - sm.start.hk * x.nt;
          break;
        }
        at += n;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;

  if (warp >= W_LOAD && warp < W_S) {
    // ---------------------------------------------------------------- producers
    // A batch of 32 pages (32 / pages-per-tile tiles): each lane holds the number and the scales of one
    // page, and fetches the next batch's while this one's loads go out.  With two loaders K and V have a
    // warp each: a lane's load takes some 100 cycles to issue.  (Where the softmax threads need more than
    // 128 registers a thirteenth warp would make them spill, which costs more: the L1 cache that would
    // hold what they spill is shared memory here.)
    constexpr int STEP = S::LOADERS;  // loads from one of this warp's to the next (K of tile j: 2 j, V: 2 j + 1)
    const int kv0 = STEP == 1 ? 0 : warp - W_LOAD;
    const int ppt_log = 7 - a.ps_log, ppt = 1 << ppt_log, batch = 32 >> ppt_log, sub = lane >> ppt_log, pg = lane & (ppt - 1);
    struct Page {
      int page, hk, active;
      float ks, vs;
    };
    Walker<R> wk;
    wk.begin(sm.start, my_tiles);
    int at = sub;  // this lane's tile in the CTA's range
    auto fetch = [&](Page& x) {
      x.active = 0;
      x.page = 0;
      x.hk = 0;
      if (at < my_tiles) {
        wk.settle(a);
        const int pos = (wk.e.t0 + wk.e.nt - 1 - wk.off) * kTile + (pg << a.ps_log);
        x.hk = wk.hk;
        x.active = pos <= wk.e.hi && pos + (1 << a.ps_log) > wk.e.lo;
        if (x.active) x.page = __ldg(a.table + (int64_t)wk.e.b * a.table_stride + (pos >> a.ps_log));
      }
      at += batch;
      wk.off += batch;
    };
    auto fetch_scales = [&](Page& x) {
      x.ks = -INFINITY;
      x.vs = 1.f;
      if (kv0 == 0 && x.active && (unsigned)x.page < (unsigned)a.num_pages) {
        if constexpr (ES == 1) {
          x.ks = __ldg(a.k_scale + (int64_t)x.page * a.Hkv + x.hk);
          x.vs = __ldg(a.v_scale + (int64_t)x.page * a.Hkv + x.hk);
        } else {
          x.ks = 1.f;
        }
      }
    };
    int issued = kv0, slot = kv0 % NS;  // load number and its slot
    uint32_t phase = 1;               // parity of the empty barriers' phase that frees it (the first is free)
    Page x, y;
    wk.off += sub;
    fetch(x);
    fetch_scales(x);
    bool ok = true;
    for (int j0 = 0; ok && j0 < my_tiles; j0 += batch) {
      fetch(y);
      const bool hidden = x.active && (unsigned)x.page >= (unsigned)a.num_pages;
      const unsigned act = __ballot_sync(0xffffffffu, x.active), hid = __ballot_sync(0xffffffffu, hidden);
      if (hid && lane == 0) report_status(a.status, FA_ERR_INVALID);
      const int page = hidden ? a.num_pages : x.page;  // reads as zeros: the map's bounds check
      const int n = min(batch, my_tiles - j0);
      const unsigned pages = (1u << ppt) - 1u;
      unsigned none = 0, far = 0;  // pages without a positive value scale, with one far from 1
      uint32_t turned = 0;
      for (int k = 0; k < n; ++k) {
        const uint32_t bytes = ((uint32_t)__popc((act >> (k << ppt_log)) & pages) << a.ps_log) * S::ROWB;
#pragma unroll
        for (int kv = kv0; kv < 2; kv += STEP) {
          ok = wait_for_w(sm.empty + slot, phase, abort_flag);
          if (!ok) break;
          uint64_t* const full = (kv ? sm.full_v : sm.full_k) + slot;
          if (lane == 0) mbar_expect_tx(full, bytes);
          __syncwarp();
          if (sub == k && x.active) {
            unsigned char* dst = base + (size_t)slot * S::SLOT + (size_t)(pg << a.ps_log) * SW;
#pragma unroll
            for (int p = 0; p < S::ROWB / SW; ++p)
              tma_load_4d(dst + p * S::PANEL, kv ? &tv : &tk, full, p * (SW / ES), 0, x.hk, page);
          }
          if (kv == 0) {
            // The scales are there before the slot's barrier can complete.  Their place in the ring is
            // free: the tile that used it lies further back than the ring of slots reaches.
            const int ring = (j0 + k) % kScaleRing;
            if (ES == 1 && k == 0) {
              const bool positive = x.vs > kNoScale && x.vs < INFINITY, some = fabsf(x.vs) > kNoScale && fabsf(x.vs) < INFINITY;
              none = __ballot_sync(0xffffffffu, x.active && !positive);
              turned = some ? kSigns : fabsf(x.vs) <= kNoScale ? kZeros : kNaNs;
              x.vs = some ? fabsf(x.vs) : kScaleless;
              far = __ballot_sync(0xffffffffu, x.active && some && !(x.vs >= 1.f / kFar2 && x.vs <= kFar2));
            }
            if (sub == k) {
              sm.scales[ring][pg] = make_float2(x.ks, x.vs);
              if (ES == 1) sm.turned[ring][pg] = none >> lane & 1u ? turned : 0u;
            }
            if (lane == 0)
              sm.odd[ring] = ((((hid | none) >> (k << ppt_log)) & pages) ? kCleared : 0) |
                             (((far >> (k << ppt_log)) & pages) ? kFar : 0);
            __syncwarp();
          }
          if (lane == 0) mbar_arrive(full);
          issued += STEP;
          slot += STEP;
          if (slot >= NS) {
            slot -= NS;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if (k == 0) fetch_scales(y);
      }
      x = y;
    }
    if (!ok && lane == 0) *abort_flag = 1;
    // Every slot's latest load lands before the CTA may exit: the last NS ones of both warps (an earlier
    // one was consumed, and its barrier has moved on).  After an abort the counts of the two warps may
    // differ, and a load that another one followed is not to be waited for: a few polls each instead.
    const int end = 2 * my_tiles;
    for (int ld = issued - STEP; ld >= 0 && ld >= (ok ? end : issued) - NS; ld -= STEP) {
      uint64_t* const full = (ld & 1 ? sm.full_v : sm.full_k) + ld % NS;
      const uint32_t parity = (uint32_t)(((ld >> 1) / turn) & 1);
      if (ok) {
        if (!wait_for_w(full, parity, never) && lane == 0) *abort_flag = 1;
      } else {
        for (int n = 0; n < 1000 && !mbar_try_wait(full, parity); ++n) __nanosleep(1000);
        __syncwarp();
      }
    }
  } else if (warp == W_S) {
    // ---------------------------------------------------------------- S issue
    // S(j) goes into buffer j & 1 once the softmax of j - 2 has read it (it has written P(j - 2)).
    const uint32_t slot_k = (uint32_t)make_smem_desc(smem_u32(base), 16, 8 * SW, LAYOUT);
    const uint32_t q_lo = (uint32_t)make_smem_desc(smem_u32(sQ), 16, 8 * SW, LAYOUT);
    const uint32_t hi_k = (uint32_t)(make_smem_desc(0, 16, 8 * SW, LAYOUT) >> 32);
    int slot = 0, j = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int seg = 0; ok && j < my_tiles; ++seg) {
      ok = wait_for_w(sm.q_full + (seg & 1), (uint32_t)((seg >> 1) & 1), abort_flag);
      const int nt = ok ? sm.rc[seg & 1].sg.nt : 0;
      const uint32_t qb = q_lo + (uint32_t)(((seg & 1) * S::QBUF) >> 4);
      for (int it = 0; ok && it < nt; ++it, ++j) {
        if (j >= 2) ok = wait_for_w(sm.p_full + (j & 1), (uint32_t)(((j >> 1) - 1) & 1), abort_flag);
        ok = ok && wait_for_w(sm.full_k + slot, phase, abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t ka = slot_k + (uint32_t)((slot * S::SLOT) >> 4);
#pragma unroll
        for (int pt = 0; pt < S::PARTS; ++pt)
#pragma unroll
          for (int kk = 0; kk < S::ROWB / 32; ++kk) {
            const uint32_t p = kk * 32 / SW, in = (kk * 32 % SW) >> 4;
            const uint32_t ad = ka + p * (S::PANEL >> 4) + in,
                           bd = qb + pt * (S::QPART >> 4) + p * (S::QPANEL >> 4) + in;
            if constexpr (ES == 1) mma_f8_ss_w(tmem + (j & 1) * N, ad, hi_k, bd, hi_k, IDESC_S, pt + kk > 0);
            else mma_ss_w(tmem + (j & 1) * N, ad, hi_k, bd, hi_k, IDESC_S, kk > 0);
          }
        tc_commit_w(sm.s_full + (j & 1));
        tc_commit_w(sm.empty + slot);
        slot += 2;
        if (slot >= NS) slot -= NS;
        if (slot == 0) phase ^= 1u;
      }
      tc_commit_w(sm.q_empty + (seg & 1));
    }
    if (!ok && lane == 0) *abort_flag = 1;
    tc_commit_w(sm.fin_bar);
    if (!wait_for_w(sm.fin_bar, 0, never) && lane == 0) *abort_flag = 1;  // every MMA has retired before TMEM is freed
  } else if (warp == W_PV) {
    // ---------------------------------------------------------------- P V issue
    // V as the M-major operand: panels of SW bytes of D are LBO apart (a head dim of 64 has one
    // panel, read twice: rows 64-127 of O repeat rows 0-63 and are not used)
    constexpr uint32_t V_LBO = D * ES > SW && ES == 2 ? S::PANEL : 0;
    const uint32_t slot_v = (uint32_t)make_smem_desc(smem_u32(base), V_LBO, 8 * SW, LAYOUT);
    const uint32_t hi_v = (uint32_t)(make_smem_desc(0, V_LBO, 8 * SW, LAYOUT) >> 32);
    // P: 16 bytes of N x 8 positions are contiguous; the next 8 positions are 128 bytes on, the
    // next 16 bytes of N 2048
    const uint32_t p_lo = (uint32_t)make_smem_desc(smem_u32(sP), 128, 2048, SMEM_SWIZZLE_NONE);
    const uint32_t hi_p = (uint32_t)(make_smem_desc(0, 128, 2048, SMEM_SWIZZLE_NONE) >> 32);
    int slot = 1 % NS, j = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int seg = 0; ok && j < my_tiles; ++seg) {
      ok = wait_for_w(sm.q_full + (seg & 1), (uint32_t)((seg >> 1) & 1), abort_flag);
      const int nt = ok ? sm.rc[seg & 1].sg.nt : 0;
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.q_empty + (seg & 1));
      // the unit before last, which used the same O, has been written
      if (TURNS && seg >= 2) ok = ok && wait_for_w(sm.done + (seg & 1), (uint32_t)(((seg >> 1) - 1) & 1), abort_flag);
      for (int it = 0; ok && it < nt; ++it, ++j) {
        ok = wait_for_w(sm.full_v + slot, phase, abort_flag) &&
             wait_for_w(sm.p_full + (j & 1), (uint32_t)((j >> 1) & 1), abort_flag);
        if (!ok) break;
        tc_fence_after();
        const uint32_t acc0 = it >= (TURNS ? 2 : 1) ? 1u : 0u;  // the first tile that this O takes overwrites it
        const uint32_t o = tmem + S::TM_O + (TURNS ? ((seg & 1) * 2 + (j & 1)) * S::ON : 0);
        const uint32_t pb = p_lo + (uint32_t)(((j & 1) * S::PBUF) >> 4);
#pragma unroll
        for (int db = 0; db < S::NO; ++db) {
          const uint32_t va = slot_v + (uint32_t)((slot * S::SLOT + db * (128 * ES / SW) * S::PANEL) >> 4);
#pragma unroll
          for (int pt = 0; pt < S::PARTS; ++pt)
#pragma unroll
            for (int kk = 0; kk < kTile / KPOS; ++kk) {
              const uint32_t ad = va + kk * ((KPOS * SW) >> 4),
                             bd = pb + pt * (S::PPART >> 4) + kk * ((KPOS * 16) >> 4);
              if constexpr (ES == 1) mma_f8_ss_w(o + db * N, ad, hi_v, bd, hi_p, IDESC_PV, pt + kk > 0 ? 1u : acc0);
              else mma_ss_w(o + db * N, ad, hi_v, bd, hi_p, IDESC_PV, kk > 0 ? 1u : acc0);
            }
        }
        tc_commit_w(sm.o_full + (j & 1));
        tc_commit_w(sm.empty + slot);
        slot += 2;
        if (slot >= NS) slot -= NS;
        if (slot == 1 % NS) phase ^= 1u;
      }
    }
    if (!ok && lane == 0) *abort_flag = 1;
    tc_commit_w(sm.fin_bar + 1);
    if (!wait_for_w(sm.fin_bar + 1, 0, never) && lane == 0) *abort_flag = 1;
  } else if (warp == W_Q) {
    // ---------------------------------------------------------------- Q operand and row constants
    // The softmax warps build the first unit's (they have nothing else to do yet).
    Walker<R> wk;
    wk.begin(sm.start, my_tiles);
    Seg sg;
    bool ok = true;
    for (int seg = 0; ok && wk.next(a, &sg); ++seg) {
      const int buf = seg & 1;
      if (seg >= 2) ok = mbar_wait_w(sm.q_empty + buf, (uint32_t)(((seg >> 1) - 1) & 1), abort_flag);
      if (!ok) break;
      if (lane == 0) sm.rc[buf].sg = sg;
      if (seg == 0) {
        bar_sync_w(6, NSM + 32);
      } else {
        build_rows<R>(a, wk.e, sg.hk, sm.rc[buf], lane, 32);
        __syncwarp();
        build_q<D, ES, R, 32>(a, sQ + buf * S::QBUF, sm.rc[buf], lane);
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.q_full + buf);
    }
    if (!ok && lane == 0) *abort_flag = 1;
  } else {
    // ---------------------------------------------------------------- softmax (thread = position)
    const int grp = warp >> 2, t = tid & 127, bar = 1 + grp;
    RowState& rs = sm.rs[grp];
    const int set = TURNS ? grp / S::H : 0, half = grp - set * S::H;
    const int c0 = half * C;  // this thread's rows are [c0, c0 + C)
    const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool capped = (a.score.flags & FA_SCORE_SOFTCAP) != 0, alibi = (a.score.flags & FA_SCORE_ALIBI) != 0;
    const float cap2 = capped ? a.score.softcap * kLog2e : 0.f, cap_k = capped ? 2.f * kLog2e / a.score.softcap : 0.f;
    const int my_page = t >> a.ps_log;
    constexpr float LIFT = lift_of(ES), SLACK = slack_of(ES), HEAD = head_of(ES);
    constexpr int PW = 16 / ES;  // rows per 16-byte store of P
    constexpr bool KEEP = R <= 16;
    constexpr bool SKIP = R <= 16;  // (elsewhere the branches cost more than the rows that they would spare)
    constexpr int CH = 4;        // rows worked on together; the ones behind the last real row are left out
    if (my_tiles > 0) {
      build_rows<R>(a, sm.start.e, sm.start.hk, sm.rc[0], tid, NSM);
      bar_sync_w(5, NSM);
      build_q<D, ES, R, NSM>(a, sQ, sm.rc[0], tid);
      fence_proxy_async_smem();
      bar_sync_w(6, NSM + 32);
    }
    int j = 0;
    uint32_t posts = 0;  // parity of the next phase of the `posted` barriers, one bit each
#pragma unroll 1
    for (int seg = 0; j < my_tiles; ++seg) {
      const RowConst<R>& rc = sm.rc[seg & 1];
      if (t < C) {
        rs.m[t] = kUnset;
        rs.bias[t] = LIFT - kUnset;
        rs.move[t] = 1.f;
      }
      if (t == 0) rs.watch = 0u, rs.far = 0;
      // Inside a unit no wait leaves the loops: after a time-out every later wait returns at once and
      // nothing is written at the end.
      // The threads of a group agree on whether the unit is known, so that they leave together.
      const bool lost = !wait_for(sm.q_full + (seg & 1), (uint32_t)((seg >> 1) & 1), abort_flag);
      if (vote_or(bar, 128, lost)) {
        *abort_flag = 1;
        break;
      }
      const Seg sg = rc.sg;
      const int rr = min(sg.rows - c0, C);  // this thread's real rows
      float l[C], xs[C], bias[C];  // (where the threads have no registers for the constants: read per tile)
#pragma unroll
      for (int n = 0; n < C; ++n) {
        l[n] = 0.f;
        xs[n] = rc.xs[c0 + n];
        bias[n] = LIFT - kUnset;
      }
      bool filled = false;  // this group's O holds something of this unit
      uint32_t seen = 0xffffffffu;  // the last tile's RowState::seen of this warp alone
      const uint32_t t_o = t_lane + S::TM_O + (TURNS ? ((seg & 1) * 2 + set) * S::ON : 0) + c0;
      for (int it = 0; it < sg.nt; ++it, ++j) {
        if (TURNS && (j & 1) != set) continue;
        const int p0 = (sg.t0 - it) * kTile, pos = p0 + t;
        if (!wait_for(sm.s_full + (j & 1), (uint32_t)((j >> 1) & 1), abort_flag)) *abort_flag = 1;
        tc_fence_after();
        uint32_t r[16];
        tmem_ld16(t_lane + (j & 1) * N + c0, r);
        const float2 sc = sm.scales[j % kScaleRing][my_page];
        const int odd = sm.odd[j % kScaleRing];
        const bool shown = sc.x != -INFINITY;
        const float ks = ES == 1 ? (shown ? sc.x : 0.f) : 1.f;
        const float lv = ES == 1 ? lg2_approx(sc.y) : 0.f;
        const float inv_vs = ES == 1 && !odd ? ex2_approx(-lv) : 0.f;
        const bool inside = p0 >= sg.in_lo && p0 + kTile - 1 <= sg.in_hi && !(odd & kCleared);
        tmem_ld_wait();
        reg_pin(r);
        float z[C], top = -INFINITY;
#pragma unroll
        for (int c = 0; c < C; c += CH) {
          if (SKIP && c >= rr) {
#pragma unroll
            for (int n = c; n < c + CH; ++n) z[n] = -INFINITY;
            continue;
          }
          if constexpr (!KEEP) {
            const float4 k4 = *reinterpret_cast<const float4*>(rc.xs + c0 + c);
            xs[c] = k4.x, xs[c + 1] = k4.y, xs[c + 2] = k4.z, xs[c + 3] = k4.w;
          }
#pragma unroll
          for (int n = c; n < c + CH; ++n) {
            float x = __uint_as_float(r[n]);
            if constexpr (S::SIDE) x += __uint_as_float(r[8 + n]);
            const float k = ES == 1 ? ks * xs[n] : xs[n];
            if constexpr (!MODS) {
              z[n] = ES == 1 ? fmaf(x, k, lv) : x * k;
            } else {
              x *= k;
              if (alibi) x = fmaf(rc.slope[c0 + n], (float)(pos - rc.qpos[c0 + n]), x);
              // cap tanh(x / cap) = cap (1 - 2 / (1 + e^(2 x / cap))), in log2 units
              if (capped) x = fmaf(-2.f * cap2, __fdividef(1.f, 1.f + ex2_approx(x * cap_k)), cap2);
              z[n] = x + lv;
            }
          }
        }
        if (!inside) {
#pragma unroll
          for (int n = 0; n < C; ++n)
            if (!shown | (pos < rc.lo[c0 + n]) | (pos > rc.hi[c0 + n])) z[n] = -INFINITY;
        }
#pragma unroll
        for (int c = 0; c < C; c += CH) {
          if (SKIP && c >= rr) continue;
          if constexpr (!KEEP) {
            const float4 b4 = *reinterpret_cast<const float4*>(rs.bias + c);
            bias[c] = b4.x, bias[c + 1] = b4.y, bias[c + 2] = b4.z, bias[c + 3] = b4.w;
          }
          top = fmax3f(top, fmax3f(z[c] + bias[c], z[c + 1] + bias[c + 1], z[c + 2] + bias[c + 2]), z[c + 3] + bias[c + 3]);
        }
        bool moves = vote_or(bar, 128, top > LIFT + SLACK);
        uint32_t low = 0;  // rows whose largest probability in both of the group's last two tiles was below 1/2
        if constexpr (ES == 1) {
          if (filled) {
            const uint4 s = rs.seen[((j >> TURNS) & 1) ^ 1];
            low = rs.watch & ~(s.x | s.y | s.z | s.w);
            moves |= low != 0;
          }
        }
        if (moves) {
          // ---- a reference has to move to the tile's largest z of its row
#pragma unroll
          for (int c = 0; c < C; c += CH) {
            if (SKIP && c >= rr) continue;
#pragma unroll
            for (int n = c; n < c + CH; ++n) {
              const float m = warp_max(z[n]);
              if (lane == n) reinterpret_cast<float*>(&rs.red[n])[warp & 3] = m;
            }
          }
          bar_sync_w(bar, 128);
          uint32_t may = 0;
          if (t < (SKIP ? (rr + CH - 1) & -CH : C)) {  // (rows worked on, real or not: an unset one would ask to move again)
            const float old = rs.m[t];
            const float4 w = rs.red[t];
            const float nm = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w));
            float m = nm > old + SLACK ? nm + HEAD : old;
            if constexpr (ES == 1) {
              float high = old == kUnset ? kUnset : rs.high[t];
              if (m == old && (low & row_bit(t))) m = fmaxf(fminf(old, nm + HEAD), high - kDrop);
              rs.high[t] = high = fmaxf(high, m);
              if (t < rr && rc.lo[c0 + t] <= rc.hi[c0 + t] && m > fmaxf(high - kDrop, kUnset)) may = row_bit(t);
            }
            rs.move[t] = m != old ? ex2_approx(old - m) : 1.f;
            rs.m[t] = m;
            rs.bias[t] = LIFT - m;
          }
          if (ES == 1 && (warp & 3) == 0) {
            may = __reduce_or_sync(0xffffffffu, may);
            if (lane == 0) rs.watch = rs.far ? 0u : may;
          }
          bar_sync_w(bar, 128);
#pragma unroll
          for (int c = 0; c < C; c += CH) {
            if (SKIP && c >= rr) continue;
            const float4 mv = *reinterpret_cast<const float4*>(rs.move + c);
            const float4 b4 = *reinterpret_cast<const float4*>(rs.bias + c);
            l[c] *= mv.x, l[c + 1] *= mv.y, l[c + 2] *= mv.z, l[c + 3] *= mv.w;
            bias[c] = b4.x, bias[c + 1] = b4.y, bias[c + 2] = b4.z, bias[c + 3] = b4.w;
          }
          if (filled) {  // this O's last P V must have retired
            const int jo = j - (TURNS ? 2 : 1);
            if (!wait_for(sm.o_full + (jo & 1), (uint32_t)((jo >> 1) & 1), abort_flag)) *abort_flag = 1;
            tc_fence_after();
#pragma unroll 1
            for (int db = 0; db < S::NO; ++db) {
              uint32_t o[16];
              tmem_ld16(t_o + db * N, o);
              tmem_ld_wait();
              reg_pin(o);
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * rs.move[k % C]);
              tmem_st16(t_o + db * N, o);
            }
            tmem_st_wait();
          }
        }
        filled = true;
        if (ES == 1 && odd) {
          const float lv = lg2_approx(sm.scales[j % kScaleRing][my_page].y);  // (read again: registers)
#pragma unroll
          for (int n = 0; n < C; ++n) l[n] += ex2_approx(z[n] - lv + (KEEP ? bias[n] : rs.bias[n]));
          if (t == 0 && (odd & kFar)) rs.far = 1, rs.watch = 0u;  // (the next vote shows it)
        }
        // P(j - 2), which lies where P(j) goes, has been read
        if (j >= 2 && !wait_for(sm.o_full + (j & 1), (uint32_t)(((j >> 1) - 1) & 1), abort_flag)) *abort_flag = 1;
        // ---- probabilities: the sum in fp32, P into shared memory as the B operand
        unsigned char* pw = sP + (j & 1) * S::PBUF + (c0 / PW) * 2048 + (t >> 3) * 128 + (t & 7) * 16;
        uint32_t hi[C / 4 * ES], lo[C / 4];  // packed P (bf16: hi alone)
#pragma unroll
        for (int c = 0; c < C; c += CH) {
#pragma unroll
          for (int k = 0; k < ES; ++k) hi[c / 4 * ES + k] = 0u;
          lo[c / 4] = 0u;
          if (SKIP && c >= rr) continue;
          if constexpr (!KEEP) {
            const float4 b4 = *reinterpret_cast<const float4*>(rs.bias + c);
            bias[c] = b4.x, bias[c + 1] = b4.y, bias[c + 2] = b4.z, bias[c + 3] = b4.w;
          }
          float p[4];
#pragma unroll
          for (int u = 0; u < CH; ++u) p[u] = ex2_approx(z[c + u] + bias[c + u]);
#pragma unroll
          for (int u = 0; u < CH; ++u) l[c + u] = ES == 1 ? fmaf(p[u], inv_vs, l[c + u]) : l[c + u] + p[u];
          if constexpr (ES == 2) {
            hi[c / 2] = pack_bf16x2(p[0], p[1]);
            hi[c / 2 + 1] = pack_bf16x2(p[2], p[3]);
          } else {
            hi[c / 4] = split_e4m3x4(p, &lo[c / 4]);
          }
        }
        if constexpr (ES == 1) {
          // a code of 1/2 is 0x30; the next tile's vote shows it to the other warps
          uint32_t now = 0;
#pragma unroll
          for (int i = 0; i < C / 4; ++i) now |= ((hi[i] + 0x50505050u) & 0x80808080u) >> i;
          now = __reduce_or_sync(0xffffffffu, now);
          if (lane == 0) reinterpret_cast<uint32_t*>(&rs.seen[(j >> TURNS) & 1])[warp & 3] = now | seen;
          seen = now;
        }
        if constexpr (S::SIDE) {
          *reinterpret_cast<uint4*>(pw) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
        } else {
          *reinterpret_cast<uint4*>(pw) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if constexpr (ES == 1) *reinterpret_cast<uint4*>(pw + S::PPART) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          else *reinterpret_cast<uint4*>(pw + 2048) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
        }
        if (p0 < sg.lo || p0 + kTile - 1 > sg.hi || (odd & kCleared)) {
          // Positions that no row sees may hold anything (a zero probability times NaN is NaN), and
          // value scales of zero make no contribution: these rows of V become zero when the tile
          // has landed.  The sign of a negative scale goes to the codes, and a NaN or an infinity makes
          // them NaN.
          const int ld = 2 * j + 1, slot = ld % NS;
          if (!wait_for(sm.full_v + slot, (uint32_t)((j / turn) & 1), abort_flag)) *abort_flag = 1;
          const bool clears = half == 0;  // one group does
          const bool seen_here = pos >= sg.lo && pos <= sg.hi;
          const uint32_t change = !seen_here ? kZeros : ES == 1 ? sm.turned[j % kScaleRing][my_page] : 0u;
          if (clears && change) {
            unsigned char* v = base + (size_t)slot * S::SLOT + t * SW;
#pragma unroll 1
            for (int p = 0; p < S::ROWB / SW; ++p)
#pragma unroll
              for (int c = 0; c < SW / 16; ++c) {
                uint4* at = reinterpret_cast<uint4*>(v + p * S::PANEL + c * 16);
                const uint32_t w = change == kZeros ? 0u : change;
                uint4 x = make_uint4(w, w, w, w);
                if (ES == 1 && change == kSigns) x.x ^= at->x, x.y ^= at->y, x.z ^= at->z, x.w ^= at->w;
                *at = x;
              }
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.p_full + (j & 1));
      }
      // ---- end of the unit's part: join the threads' sums (and the groups', where they took turns),
      //      scale O and write it
      Posted& mine = sm.post[seg & 1][grp];
      const bool both = TURNS && sg.nt >= 2;               // the other set has tiles of this unit too
      const bool writer = !TURNS || ((j - 1) & 1) == set;  // this one has the last tile
      if (writer || both) {
        if (both && !writer && seg >= 2 &&  // what was posted two units ago has been read
            !wait_for(sm.done + (seg & 1), (uint32_t)(((seg >> 1) - 1) & 1), abort_flag))
          *abort_flag = 1;
        const float ls = warp_col_sums<C>(l, lane);
        if (lane % (32 / C) == 0) reinterpret_cast<float*>(&mine.sum[lane / (32 / C)])[warp & 3] = ls;
        if (t < C) mine.m[t] = rs.m[t];
        if (!writer) {
          __syncwarp();
          if (lane == 0) mbar_arrive(sm.posted + (seg & 1));
        }
      }
      if (writer) {
        bar_sync_w(bar, 128);
        if (both && !wait_for(sm.posted + (seg & 1), (posts >> (seg & 1)) & 1u, abort_flag)) *abort_flag = 1;
        const bool whole = sg.first && sg.last;
        const int part = 2 * cta + (seg == 0 ? 0 : 1);
        if (t == 0 && half == 0 && sg.first && !sg.last) {  // the CTA's last unit, which goes on in the next CTAs
          const int end = my_start + my_tiles - sg.nt + sg.entry_nt;
          sm.join_parts = (end - 1) / per - cta + 1;
          sm.join_slot = part;
          sm.join_entry = sg.entry;
          sm.join_hk = sg.hk;
        }
        if (t < C) {
          const float4 w = mine.sum[t];
          float m = mine.m[t], sum = (w.x + w.y) + (w.z + w.w), f = 1.f, fo = 0.f;
          if (both) {  // the other set's partial sums, references and O
            const Posted& other = sm.post[seg & 1][(set ^ 1) * S::H + half];
            const float4 wo = other.sum[t];
            const float mo = other.m[t], so = (wo.x + wo.y) + (wo.z + wo.w), top = fmaxf(m, mo);
            f = ex2_approx(m - top);
            fo = ex2_approx(mo - top);
            sum = sum * f + so * fo;
            m = top;
          }
          // a NaN stays one; a row that may see nothing took part in the tiles that needed no mask
          const bool some = !(sum == 0.f) && rc.lo[c0 + t] <= rc.hi[c0 + t];
          const float inv = some ? (ES == 1 ? 0x1p-8f : 1.f) / sum : 0.f;  // (8-bit P is 2^8 times what the sum adds)
          rs.fin[0][t] = some ? f * inv : -1.f;  // negative: zeros, whatever O holds (0 times a NaN is one)
          rs.fin[1][t] = fo * inv;
          const float lse = some ? (m - LIFT + lg2_approx(sum)) * kLn2 : -INFINITY;
          if (!*abort_flag) {
            if (!whole) a.part_lse[(int64_t)part * R + c0 + t] = lse;
            else if (t < rr) a.lse[rc.lrow[c0 + t]] = lse;
          }
        }
        // The last P V, and so all before it (one thread's MMAs end in order).
        if (!wait_for(sm.o_full + ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag)) *abort_flag = 1;
        tc_fence_after();
        bar_sync_w(bar, 128);
        const bool good = !__any_sync(0xffffffffu, *abort_flag);
        if (D >= 128 || (warp & 3) < 2) {
          const uint32_t t_other = t_lane + S::TM_O + ((seg & 1) * 2 + (set ^ 1)) * S::ON + c0;
#pragma unroll 1
          for (int n0 = 0; n0 < rr; n0 += 4)
#pragma unroll 1
            for (int db = 0; db < S::NO; ++db) {
              const int d = db * 128 + t, at = db * N + n0;
              uint32_t x[4], y[4] = {}, x2[4] = {}, y2[4] = {};
              tmem_ld4(t_o + at, x);
              if constexpr (S::SIDE) tmem_ld4(t_o + at + 8, y);
              if (both) {
                tmem_ld4(t_other + at, x2);
                if constexpr (S::SIDE) tmem_ld4(t_other + at + 8, y2);
              }
              tmem_ld_wait();
              reg_pin(x);
              reg_pin(y);
              reg_pin(x2);
              reg_pin(y2);
              if (!good) continue;
              const float4 f4 = *reinterpret_cast<const float4*>(rs.fin[0] + n0), g4 = *reinterpret_cast<const float4*>(rs.fin[1] + n0);
              const float f[4] = {f4.x, f4.y, f4.z, f4.w}, g[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int n = c0 + n0 + u;
                float v = __uint_as_float(x[u]), o = __uint_as_float(x2[u]);
                if constexpr (S::SIDE) {
                  v += __uint_as_float(y[u]);
                  o += __uint_as_float(y2[u]);
                }
                v *= f[u];
                if constexpr (TURNS) v = fmaf(o, g[u], v);
                if (f[u] < 0.f) v = 0.f;
                if (!whole) a.part_o[((int64_t)part * R + n) * D + d] = v;
                else if (n0 + u < rr) reinterpret_cast<__nv_bfloat16*>(a.o.ptr)[rc.orow[n] + d] = __float2bfloat16_rn(v);
              }
            }
        }
        tc_fence_before();
      }
      if (both) posts ^= 1u << (seg & 1);
      __syncwarp();
      if (lane == 0) {
        if (TURNS && writer) mbar_arrive(sm.done + (seg & 1));
        mbar_arrive(sm.q_empty + (seg & 1));
      }
      // The references are set anew when all of their readers are here.
      bar_sync_w(bar, 128);
    }
  }
  tc_fence_before();
  __syncthreads();
  // every warp's waits are behind: one that gave up shows here, whichever it was
  if (tid == 0 && *abort_flag) report_status(a.status, FA_ERR_TIMEOUT);
  if (warp == W_S) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, S::TM_COLS);
  }
  // ---------------------------------------------------------------- entries without a tile: rows that see nothing
  // Head hk of entry e is CTA (e + hk) % CTAs's.
  const int noted = min(sm.empties, 64);
  for (int k = 0; k < noted; ++k) empty_rows<D, R>(a, sm.empty_entry[k], cta, warp, NT / 32, lane);
  if (sm.empties > 64)  // more than the list holds: look again
    for (int e = 0; e < a.entries; ++e)
      if (entry_of<R>(a, e).nt == 0) empty_rows<D, R>(a, e, cta, warp, NT / 32, lane);
  if (!a.joins) return;
  // ---------------------------------------------------------------- units that cross CTAs
  const auto grid = cooperative_groups::this_grid();
  auto arrived = grid.barrier_arrive();
  const int parts = sm.join_parts;
  if (!parts || *abort_flag) return;
  const int hk = sm.join_hk, slot0 = sm.join_slot, en = sm.join_entry, b = a.groups == 1 ? en : en / a.groups,
            m0 = (en - b * a.groups) * R;
  grid.barrier_wait(static_cast<decltype(arrived)&&>(arrived));
  // One warp per query row, 32 parts at a time: lane k weighs part k, then every lane sums its
  // elements of D over the parts, rescaled when a later batch has a larger lse.
  for (int n = warp; n < R && m0 + n < a.M; n += NT / 32) {
    float acc[D / 32], top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
    float po[8][D / 32];
    auto fetch = [&](int k, int many) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int v = 0; v < D / 32; ++v)
          po[i][v] = i < many
                         ? __ldcg(a.part_o + ((int64_t)(k + i == 0 ? slot0 : 2 * (cta + k + i)) * R + n) * D + lane + 32 * v)
                         : 0.f;
    };
#pragma unroll 1
    for (int k0 = 0; k0 < parts; k0 += 32) {
      const int k = k0 + lane, run = min(32, parts - k0);
      fetch(k0, min(8, run));  // together with the lse
      const float ls = lane < run ? __ldcg(a.part_lse + (int64_t)(k == 0 ? slot0 : 2 * (cta + k)) * R + n) : -INFINITY;
      const float nt = fmaxf(top, warp_max(ls)), ref = nt == -INFINITY ? 0.f : nt;
      const float w = lane < run ? expf(ls - ref) : 0.f;
      float ws = w;
#pragma unroll
      for (int o = 16; o; o >>= 1) ws += __shfl_xor_sync(0xffffffffu, ws, o);
      const float back = top == -INFINITY ? 0.f : expf(top - ref);
      sum = sum * back + ws;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] *= back;
      top = nt;
#pragma unroll 1
      for (int i0 = 0; i0 < run; i0 += 8) {
        if (i0 > 0) fetch(k0 + i0, min(8, run - i0));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float wi = __shfl_sync(0xffffffffu, w, i0 + i);  // (0 behind the last part)
#pragma unroll
          for (int v = 0; v < D / 32; ++v) acc[v] = fmaf(wi, po[i][v], acc[v]);
        }
      }
    }
    const int m = m0 + n, i = m / a.G, h = hk * a.G + m - i * a.G;
    __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.o.ptr) + (int64_t)b * a.o.stride_b +
                       (int64_t)h * a.o.stride_h + (int64_t)i * a.o.stride_t;
    const bool some = !(sum == 0.f);
    const float inv = some ? 1.f / sum : 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[lane + 32 * k] = __float2bfloat16_rn(acc[k] * inv);
    if (lane == 0) a.lse[((int64_t)b * a.H + h) * a.Tq + i] = some ? (top == -INFINITY ? 0.f : top) + logf(sum) : -INFINITY;
  }
}

// SMs of the current device, each of which takes one CTA (148 where there is no device to ask).
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    n = 0;
  return n > 0 ? n : 148;
}

struct PagedPlan {
  int R, groups, ctas;
  size_t workspace;
};

// Rows per group: the smallest operand width that holds every query row of a K/V head, or 64 with as
// many groups as it takes, each reading the cache again.  32 instead of 64 where bf16 pages of head dim
// 256 leave no room for more, and where the table's whole width makes at most eight tiles of 64 rows an SM:
// there the latency of a unit counts, not the cache's bytes.  Measured with 32 against 64 rows (8-bit, D 128,
// 64 query rows a K/V head, four users; us by tiles an SM): 0.9: 15 / 17, 1.7: 18 / 19, 3.5: 25 / 22, 6.9: 30 / 35,
// 13.8: 42 / 44, 28: 69 / 62, 55: 119 / 93; bf16 and head dims 64 and 256 cross between 7 and 28 as well.  The
// lengths are on the device, so short sequences in a wide table get the 64 rows.
PagedPlan plan_paged(const FaPagedAttnParams* p) {
  PagedPlan pl;
  const bool f8 = p->cache.dtype == FA_DTYPE_E4M3;
  const int sms = sm_count();
  const int64_t M = (int64_t)(p->H / p->cache.H_kv) * p->Tq;
  const int64_t tiles = (int64_t)p->B * p->cache.H_kv *
                        (((int64_t)p->cache.table_cols * p->cache.page_size + kTile - 1) / kTile);  // of one row group
  pl.R = f8 ? 8 : 16;
  while (pl.R < M && pl.R < 64) pl.R *= 2;
  if (pl.R == 64 && ((!f8 && p->cache.D == 256) || tiles * ((M + 63) / 64) <= (int64_t)8 * sms)) pl.R = 32;
  pl.groups = (int)((M + pl.R - 1) / pl.R);
  pl.ctas = (int)std::min<int64_t>(sms, tiles * pl.groups);
  pl.workspace = (size_t)2 * pl.ctas * pl.R * (p->cache.D + 1) * 4 + 256;
  return pl;
}

int check_paged(const FaPagedAttnParams* p) {
  if (!p) return set_last_error(FA_ERR_INVALID, "fa_paged_attn: params is NULL");
  int rc = check_paged_cache(p->cache, p->B, "fa_paged_attn");
  if (rc) return rc;
  if (p->H <= 0 || p->Tq <= 0) return set_last_error(FA_ERR_INVALID, "fa_paged_attn: non-positive shape (H or Tq)");
  if (p->H % p->cache.H_kv) return set_last_error(FA_ERR_INVALID, "fa_paged_attn: H must be a multiple of H_kv");
  if (p->mask.flags & ~(FA_MASK_CAUSAL | FA_MASK_WINDOW))
    return set_last_error(FA_ERR_UNSUPPORTED, "fa_paged_attn: only causal and sliding-window masks");
  if (p->mask.q_offset || p->mask.kv_offset)
    return set_last_error(FA_ERR_INVALID, "fa_paged_attn: positions come from kv_lens; offsets must be 0");
  if (p->score.flags & ~(FA_SCORE_ALIBI | FA_SCORE_SOFTCAP))
    return set_last_error(FA_ERR_UNSUPPORTED, "fa_paged_attn: only ALiBi and softcap score mods");
  if ((p->score.flags & FA_SCORE_ALIBI) && !p->score.alibi_slopes)
    return set_last_error(FA_ERR_INVALID, "fa_paged_attn: ALiBi without slopes");
  if ((p->score.flags & FA_SCORE_SOFTCAP) && !(p->score.softcap > 0.f))
    return set_last_error(FA_ERR_INVALID, "fa_paged_attn: softcap must be > 0");
  const int64_t M = (int64_t)(p->H / p->cache.H_kv) * p->Tq;
  const int64_t groups = (M + 15) / 16 + 1;
  if (M >= (1 << 30) || (int64_t)p->B * groups * p->cache.H_kv *
                                (((int64_t)p->cache.table_cols * p->cache.page_size + kTile - 1) / kTile) >=
                            (int64_t)1 << 30)
    return set_last_error(FA_ERR_UNSUPPORTED, "fa_paged_attn: too many query rows and cached positions for one call");
  return FA_OK;
}

template <int D, int ES, int R, bool MODS>
cudaError_t launch_paged(const CUtensorMap& tk, const CUtensorMap& tv, PagedArgs& a, const PagedPlan& pl,
                         cudaStream_t stream) {
  const size_t fixed = paged_smem_bytes<D, ES, R>(0), limit = 232448;
  // (two loaders: 6, 13 or 24; an odd ring below 9 would let one take a slot by the parity of its last use but one)
  a.slots = (int)std::min<size_t>(kMaxSlots, (limit - fixed) / Shape<D, ES, R>::SLOT);
  const size_t smem = paged_smem_bytes<D, ES, R>(a.slots);
  cudaError_t e =
      cudaFuncSetAttribute(paged_attn_kernel<D, ES, R, MODS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  a.joins = (a.cols << a.ps_log) > kTile && pl.ctas > 1;  // (a unit of one tile lies in one CTA)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)pl.ctas);
  cfg.blockDim = dim3(Shape<D, ES, R>::NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeCooperative;
  at.val.cooperative = a.joins;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attn_kernel<D, ES, R, MODS>, tk, tv, (const PagedArgs)a);
}

template <int D, int ES, int R>
cudaError_t launch_mods(const CUtensorMap& tk, const CUtensorMap& tv, PagedArgs& a, const PagedPlan& pl,
                        cudaStream_t st) {
  return a.score.flags ? launch_paged<D, ES, R, true>(tk, tv, a, pl, st) : launch_paged<D, ES, R, false>(tk, tv, a, pl, st);
}

template <int D>
cudaError_t launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, PagedArgs& a, const PagedPlan& pl, bool f8,
                        cudaStream_t st) {
  if (f8) {
    switch (pl.R) {
      case 8: return launch_mods<D, 1, 8>(tk, tv, a, pl, st);
      case 16: return launch_mods<D, 1, 16>(tk, tv, a, pl, st);
      case 32: return launch_mods<D, 1, 32>(tk, tv, a, pl, st);
      default: return launch_mods<D, 1, 64>(tk, tv, a, pl, st);
    }
  }
  if (pl.R == 16) return launch_mods<D, 2, 16>(tk, tv, a, pl, st);
  if (D == 256 || pl.R == 32) return launch_mods<D, 2, 32>(tk, tv, a, pl, st);
  if constexpr (D < 256) return launch_mods<D, 2, 64>(tk, tv, a, pl, st);
  return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace fa

extern "C" {

int fa_paged_attn_workspace_size(const FaPagedAttnParams* p, size_t* bytes) {
  int rc = fa::check_paged(p);
  if (rc) return rc;
  if (!bytes) return fa::set_last_error(FA_ERR_INVALID, "fa_paged_attn_workspace_size: bytes is NULL");
  *bytes = fa::plan_paged(p).workspace;
  return FA_OK;
}

int fa_paged_attn(const FaPagedAttnParams* p, void* workspace, size_t workspace_bytes, fa_stream_t stream) {
  int rc = fa::check_paged(p);
  if (rc) return rc;
  if (!p->q.ptr || !p->o.ptr || !p->lse || !p->kv_lens)
    return fa::set_last_error(FA_ERR_INVALID, "fa_paged_attn: NULL tensor");
  const fa::PagedPlan pl = fa::plan_paged(p);
  char msg[192];
  if (!workspace || workspace_bytes < pl.workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u)) {
    snprintf(msg, sizeof(msg), "fa_paged_attn: workspace must be 16-byte aligned and hold %zu bytes", pl.workspace);
    return fa::set_last_error(FA_ERR_INVALID, msg);
  }
  const FaPagedCache& c = p->cache;
  CUtensorMap tk, tv;
  if ((rc = fa::make_page_map(&tk, c, c.k, "the key pages")) || (rc = fa::make_page_map(&tv, c, c.v, "the value pages")))
    return rc;
  fa::PagedArgs a;
  a.B = p->B;
  a.H = p->H;
  a.Hkv = c.H_kv;
  a.Tq = p->Tq;
  a.G = p->H / c.H_kv;
  a.M = a.G * p->Tq;
  a.ps_log = c.page_size == 16 ? 4 : c.page_size == 32 ? 5 : c.page_size == 64 ? 6 : 7;
  a.cols = c.table_cols;
  a.num_pages = c.num_pages;
  a.groups = pl.groups;
  a.entries = p->B * pl.groups;
  a.slots = 0;
  a.q_vec = (reinterpret_cast<uintptr_t>(p->q.ptr) % 16 == 0) && p->q.stride_b % 8 == 0 && p->q.stride_h % 8 == 0 &&
            p->q.stride_t % 8 == 0;
  a.table_stride = c.table_stride;
  a.q = p->q;
  a.o = p->o;
  a.lse = p->lse;
  a.kv_lens = p->kv_lens;
  a.q_lens = p->q_lens;
  a.table = c.block_table;
  a.k_scale = c.k_scale;
  a.v_scale = c.v_scale;
  a.scale = p->scale;
  a.mask = p->mask;  // windows beyond 2^30 reach every position; cut, their sums stay within 32 bits
  a.mask.window_left = std::min(a.mask.window_left, 1 << 30);
  a.mask.window_right = std::min(a.mask.window_right, 1 << 30);
  a.score = p->score;
  a.part_o = reinterpret_cast<float*>(workspace);
  a.part_lse = a.part_o + (size_t)2 * pl.ctas * pl.R * c.D;
  a.status = p->status;
  const bool f8 = c.dtype == FA_DTYPE_E4M3;
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = c.D == 64    ? fa::launch_rows<64>(tk, tv, a, pl, f8, st)
                        : c.D == 128 ? fa::launch_rows<128>(tk, tv, a, pl, f8, st)
                                     : fa::launch_rows<256>(tk, tv, a, pl, f8, st);
  if (e != cudaSuccess) {
    snprintf(msg, sizeof(msg), "fa_paged_attn: %s", cudaGetErrorString(e));
    return fa::set_last_error(FA_ERR_CUDA, msg);
  }
  return FA_OK;
}

}  // extern "C"
