// Attention of query rows against a paged K/V cache (fa_paged_attn), bf16 or 8-bit (e4m3).
//
// Per query row: x_j = score(scale * q . k_j), o = sum_j softmax(x)_j v_j, with k_j = ks * code and
// v_j = vs * code where ks, vs belong to the page and K/V head of position j.  A decode step reads
// every cached byte once and does a few multiply-adds with each, so HBM bounds it; a prompt
// chunk is bound by the tensor cores and the exponentials.
//
// Orientation.  The 128 cached positions of a tile are the MMA's M, the query rows its N:
//     S^T [128 positions x N] = K Q^T       A = K as stored (K-major), B = Q
//     O^T [D x N]            += V^T P^T     A = V as stored (M-major), B = P from shared memory
// so the exponentials are spent on real query rows only (N is 8 to 64 of them; with the rows as M
// they would be padded to 128), and each thread owns one position: its page's scales are two
// registers.
//
// 8-bit codes go to the tensor cores as they are (kind::f8f6f4): converting a tile in shared memory
// would cost as many instructions as everything else here.  The other operand is split into two e4m3
// parts side by side in N, z = hi + lo / 16: q is scaled by a power of two per row so that its largest
// magnitude lies in [128, 256); a bf16 has 8 significant bits, each part 4, so the split is exact
// down to 2^-20 of the row's largest element.  Probabilities lie in [0, 256] and keep a relative
// error of 2^-9 (the bf16 path rounds them to 2^-9 too); what is lost below 2^-14 of the largest
// is below the sums' own rounding.  Both products accumulate in fp32.
//
// Scales.  ks multiplies the thread's logits.  vs goes into the probabilities: P = 2^(x + log2 vs -
// my + 4) with a reference my of its own per row, so that a row whose weight sits on pages of small
// values keeps its precision.  The softmax sum uses x - mx.  Both references move only when a tile
// exceeds them by more than 4 (log2 units), one barrier vote per tile.
//
// Work.  The tiles of all (sequence, row group, K/V head) units, in that order, are cut into equal
// contiguous ranges, one per CTA (one CTA per SM): ragged batches balance themselves, and nothing
// about the lengths is needed on the host.  A unit inside one CTA is written to o directly; one
// that crosses CTAs leaves at most one partial (o, lse) at each end of a CTA's range in the
// workspace, joined by paged_merge_kernel in CTA order.
//
// Warps: 0-3 softmax (thread = position of the tile; later = element of D), 4 TMA producer (lane =
// page of the tile), 5 MMA issue, 6-7 build the next unit's Q operand and row constants.
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
constexpr int kPThreads = 256;
constexpr int kSms = 148;
constexpr int kMaxSlots = 24;      // K or V tiles in the shared-memory ring
constexpr int kScaleRing = kMaxSlots / 2 + 4;  // tiles whose scales may be live at once
constexpr float kSlack = 4.f;      // a reference moves when exceeded by this much (log2 units)
constexpr float kLift = 4.f;       // 8-bit P is 2^(x - reference + kLift) <= 2^(kSlack + kLift)

struct PagedArgs {
  int B, H, Hkv, Tq, G, M;         // M = G * Tq query rows per sequence and K/V head
  int ps, cols, num_pages, groups; // groups of R query rows per (sequence, K/V head)
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
  int32_t* part_unit;  // [2 * CTAs]: 2 * unit + (the part is the unit's first), or -1
  int* status;
};

template <int D, int ES, int R>
struct Shape {
  static constexpr int N = ES == 1 ? 2 * R : R;     // columns of S and O: hi and lo parts, or rows
  static constexpr int ROWB = D * ES;               // bytes of one cached position
  static constexpr int SW = ROWB < 128 ? 64 : 128;  // swizzle span
  static constexpr int PANEL = kTile * SW;
  static constexpr int SLOT = kTile * ROWB;
  static constexpr int QPANEL = N * SW;
  static constexpr int QBUF = N * ROWB;
  static constexpr int PBUF = N * kTile * ES;
  static constexpr int NO = D <= 128 ? 1 : D / 128; // blocks of 128 elements of O
  static constexpr uint32_t TM_O = 2 * N;           // TMEM: two S buffers, then O
  static constexpr int USED = (2 + NO) * N;
  static constexpr uint32_t TM_COLS = USED <= 32 ? 32 : USED <= 64 ? 64 : USED <= 128 ? 128 : USED <= 256 ? 256 : 512;
  static_assert(USED <= 512 && N % 16 == 0 && N <= 256, "operand shape");
};

// Row constants of one unit, built by warps 6-7 (double-buffered with Q).
template <int R> struct RowConst {
  float xs[R];      // logit = dot * (ks * xs): scale, the row's power of two, and log2(e) unless softcapped
  float slope[R];   // ALiBi slope in the same domain
  int lo[R], hi[R]; // positions the row may see; hi < lo: none
  int qpos[R];
  int64_t orow[R];  // element offset of the row in o, -1: no such row
  int64_t lrow[R];  // index of the row in lse
};
// Running state of the unit in work, and scratch of the softmax warps.
template <int R> struct RowState {
  float mx[R], my[R];          // references of the sum and of O (log2 units), -inf at first
  float mref[R], thx[R], thy[R], w[R];  // mx or 0; mx + slack; my + slack; 2^(mref - my + lift)
  float al[R], ao[R];          // factors of the last move
  float fin[R];                // factor of O at the end
  float red[4][2][R];
};
template <int R> struct Smem {
  RowConst<R> rc[2];
  RowState<R> rs;
  float2 scales[kScaleRing][8];  // (ks, vs) of a tile's pages; ks = -inf hides the page
  int odd[kScaleRing];           // the tile has a hidden page
  uint64_t full[kMaxSlots], empty[kMaxSlots], s_full[2], p_full[2], o_full[2], q_full[2], q_empty[2], fin_bar;
  int scan[8];
  int total, per_cta, first_entry, first_off;
  uint32_t tmem;
  int abort_flag, never;
};

template <int D, int ES, int R>
size_t paged_smem_bytes(int slots) {
  using S = Shape<D, ES, R>;
  return 1024 + (size_t)slots * S::SLOT + 2 * S::QBUF + 2 * S::PBUF + sizeof(Smem<R>);
}

// What one (sequence, row group) has to visit.
struct Entry {
  int b, rg, len, ql, i0, i1;  // tokens i0..i1 (clipped to the valid ones)
  int lo, hi;                  // positions that some row of the group may see
  int in_lo, in_hi;            // positions that every valid row of the group may see
  int t0, nt;                  // tiles
};

template <int R>
__device__ __forceinline__ Entry entry_of(const PagedArgs& a, int e) {
  Entry x;
  x.b = e / a.groups;
  x.rg = e - x.b * a.groups;
  const int cap = a.cols * a.ps;
  x.len = min(max(__ldg(a.kv_lens + x.b), 0), cap);
  x.ql = a.q_lens ? min(max(__ldg(a.q_lens + x.b), 0), a.Tq) : a.Tq;
  x.i0 = x.rg * R / a.G;
  x.i1 = min((min(x.rg * R + R, a.M) - 1) / a.G, x.ql - 1);
  const int p0 = x.len - x.ql + x.i0, p1 = x.len - x.ql + x.i1;  // positions of the group's rows
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
  x.nt = (x.i1 < x.i0 || x.hi < x.lo) ? 0 : x.hi / kTile - x.t0 + 1;
  return x;
}

// One CTA's range of tiles, unit by unit.  Every role walks the same sequence by itself.
struct Seg {
  int hk, t0, nt;   // K/V head, first tile (absolute), tiles
  bool first, last; // holds the unit's first / last tile
};
template <int R>
struct Walker {
  Entry e;
  int idx, hk, off, left;
  __device__ __forceinline__ void begin(const PagedArgs& a, int entry, int entry_off, int tiles) {
    left = tiles;
    idx = entry;
    hk = off = 0;
    e.nt = 0;
    if (tiles > 0) {
      e = entry_of<R>(a, entry);
      hk = entry_off / e.nt;
      off = entry_off - hk * e.nt;
    }
  }
  __device__ __forceinline__ bool next(const PagedArgs& a, Seg* s) {
    if (left <= 0) return false;
    while (off >= e.nt) {  // the unit is done: the next head, or the next entry that has tiles
      off = 0;
      if (e.nt > 0 && ++hk < a.Hkv) break;
      hk = 0;
      e = entry_of<R>(a, ++idx);
      if (e.nt > 0) break;
    }
    s->hk = hk;
    s->t0 = e.t0 + off;
    s->nt = min(e.nt - off, left);
    s->first = off == 0;
    off += s->nt;
    s->last = off == e.nt;
    left -= s->nt;
    return true;
  }
};

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

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_value(uint32_t v) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// Two values as hi + lo / 16: the packed hi parts, and the lo parts through *lo2.
__device__ __forceinline__ uint32_t split_e4m3x2(float a, float b, uint32_t* lo2) {
  const uint32_t h = e4m3x2(a, b);
  const float2 v = e4m3x2_value(h);
  *lo2 = e4m3x2((a - v.x) * 16.f, (b - v.y) * 16.f);
  return h;
}

// Byte offset of 16-byte chunk c of row r in a panel of rows of SW bytes, swizzled over SW.
template <int SW>
__device__ __forceinline__ uint32_t panel_off(int r, int c) {
  return (uint32_t)(r * SW + ((SW == 128 ? (c ^ (r & 7)) : (c ^ ((r >> 1) & 3))) << 4));
}

// Columns [c, c + W) of a TMEM row (W 16 or 32) as floats, without waiting.
template <int W>
__device__ __forceinline__ void tmem_cols(uint32_t addr, uint32_t (&r)[W]) {
  if constexpr (W == 16) tmem_ld16(addr, r);
  else tmem_ld32(addr, r);
}
template <int W>
__device__ __forceinline__ void tmem_put(uint32_t addr, const uint32_t (&r)[W]) {
  if constexpr (W == 16) tmem_st16(addr, r);
  else tmem_st32(addr, r);
}

template <int D, int ES, int R>
__global__ void __launch_bounds__(kPThreads, 1)
    paged_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                      const PagedArgs a) {
  using S = Shape<D, ES, R>;
  constexpr int N = S::N, SW = S::SW;
  constexpr uint32_t LAYOUT = SW == 128 ? SMEM_SWIZZLE_128B : SMEM_SWIZZLE_64B;
  constexpr int KPOS = 32 / ES;  // positions per PV MMA
  constexpr uint32_t IDESC_S = ES == 1 ? make_idesc_e4m3(128, N, 0, 0) : make_idesc_bf16(128, N, 0, 0);
  constexpr uint32_t IDESC_PV = ES == 1 ? make_idesc_e4m3(128, N, 1, 1) : make_idesc_bf16(128, N, 1, 1);

  extern __shared__ unsigned char dsm_raw[];
  unsigned char* base =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(dsm_raw) + 1023) & ~uintptr_t(1023));
  const int NS = a.slots;
  unsigned char* sQ = base + (size_t)NS * S::SLOT;
  unsigned char* sP = sQ + 2 * S::QBUF;
  Smem<R>& sm = *reinterpret_cast<Smem<R>*>(sP + 2 * S::PBUF);
  volatile int* abort_flag = &sm.abort_flag;
  volatile int* never = &sm.never;  // stays 0: waits on it end by time only

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, cta = blockIdx.x;
  griddep_launch();

  // ---------------------------------------------------------------- setup: barriers, TMEM, range
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(sm.full + i, 1);
      mbar_init(sm.empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(sm.s_full + i, 1);
      mbar_init(sm.p_full + i, 4);
      mbar_init(sm.o_full + i, 1);
      mbar_init(sm.q_full + i, 2);
      mbar_init(sm.q_empty + i, 5);  // the MMA issuer's commit and four softmax warps
    }
    mbar_init(&sm.fin_bar, 1);
    sm.abort_flag = 0;
    sm.never = 0;
    fence_mbar_init();
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 5) {
    tmem_alloc(&sm.tmem, S::TM_COLS);
    tmem_relinquish();
  }
  {
    // Exclusive prefix of the entries' tiles over the threads, each with a run of entries.
    const int run = (a.entries + kPThreads - 1) / kPThreads, e0 = min(tid * run, a.entries),
              e1 = min(e0 + run, a.entries);
    int mine = 0;
    bool bad = false;
    for (int e = e0; e < e1; ++e) {
      const Entry x = entry_of<R>(a, e);
      mine += x.nt * a.Hkv;
      if (x.rg == 0) {
        const int n = __ldg(a.kv_lens + x.b), t = a.q_lens ? __ldg(a.q_lens + x.b) : 0;
        bad = bad || n < 0 || n > a.cols * a.ps || t < 0 || t > a.Tq;
      }
    }
    if (bad && cta == 0) report_status(a.status, FA_ERR_INVALID);
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
    for (int w = 0; w < 8; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
    }
    const int per = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
    const int start = (int)min((int64_t)cta * per, (int64_t)total);
    int at = before + inc - mine;
    if (start < total && at <= start && start < at + mine) {
      for (int e = e0; e < e1; ++e) {
        const int n = entry_of<R>(a, e).nt * a.Hkv;
        if (start < at + n) {
          sm.first_entry = e;
          sm.first_off = start - at;
          break;
        }
        at += n;
      }
    }
    if (tid == 0) {
      sm.total = total;
      sm.per_cta = per;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;
  const int my_start = (int)min((int64_t)cta * sm.per_cta, (int64_t)sm.total);
  const int my_tiles = min(sm.per_cta, sm.total - my_start);
  Walker<R> wk;
  wk.begin(a, sm.first_entry, sm.first_off, my_tiles);
  Seg sg;

  if (warp == 4) {
    // ---------------------------------------------------------------- producer
    // Lane l serves page l of a tile.  Page numbers are fetched two tiles ahead and scales one, so
    // neither latency holds up the ring.
    const int ppt = kTile / a.ps;
    struct Ahead {
      int page, col, hk, tile, active, lo, hi;
      float ks, vs;
    };
    Ahead x0, x1, x2;  // the tile to issue, the next, the one after
    int left_in_seg = 0, tile = 0;
    auto fetch = [&](Ahead& x) {  // page number of the next tile of the walk
      x.tile = -1;
      if (left_in_seg == 0) {
        if (!wk.next(a, &sg)) return;
        left_in_seg = sg.nt;
        tile = sg.t0;
      }
      x.tile = tile++;
      --left_in_seg;
      x.hk = sg.hk;
      const int pos = x.tile * kTile + lane * a.ps;
      x.active = lane < ppt && pos <= wk.e.hi && pos + a.ps > wk.e.lo;
      x.page = x.active ? __ldg(a.table + (int64_t)wk.e.b * a.table_stride + pos / a.ps) : 0;
    };
    auto fetch_scales = [&](Ahead& x) {
      const bool good = x.tile >= 0 && x.active && (unsigned)x.page < (unsigned)a.num_pages;
      x.ks = -INFINITY;
      x.vs = 0.f;
      if (good) {
        if constexpr (ES == 1) {
          x.ks = __ldg(a.k_scale + (int64_t)x.page * a.Hkv + x.hk);
          x.vs = __ldg(a.v_scale + (int64_t)x.page * a.Hkv + x.hk);
        } else {
          x.ks = 1.f;
          x.vs = 1.f;
        }
      }
    };
    int issued = 0;  // slots filled so far (K and V of a tile take one each)
    fetch(x0);
    fetch(x1);
    fetch_scales(x0);
    for (int j = 0; x0.tile >= 0; ++j) {
      fetch(x2);
      fetch_scales(x1);
      const bool hidden = x0.active && (unsigned)x0.page >= (unsigned)a.num_pages;
      const unsigned act = __ballot_sync(0xffffffffu, x0.active);
      const bool any_hidden = __any_sync(0xffffffffu, hidden);
      if (any_hidden && lane == 0) report_status(a.status, FA_ERR_INVALID);
      const uint32_t bytes = (uint32_t)__popc(act) * a.ps * S::ROWB;
      bool ok = true;
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const int ld = 2 * j + kv, slot = ld % NS;
        if (ld >= NS) ok = mbar_wait_w(sm.empty + slot, (uint32_t)((ld / NS - 1) & 1), abort_flag);
        if (!ok) break;
        if (kv == 0) {  // the K slot's release says that the tile whose scales lay here is done
          if (lane < 8) sm.scales[j % kScaleRing][lane] = make_float2(x0.ks, x0.vs);
          if (lane == 0) sm.odd[j % kScaleRing] = any_hidden;
          __syncwarp();
        }
        if (lane == 0) mbar_arrive_expect_tx(sm.full + slot, bytes);
        __syncwarp();
        if (x0.active) {  // a page number out of range reads as zeros: the map's bounds check
          unsigned char* dst = base + (size_t)slot * S::SLOT + (size_t)lane * a.ps * SW;
          const int page = hidden ? a.num_pages : x0.page;
#pragma unroll
          for (int p = 0; p < S::ROWB / SW; ++p)
            tma_load_4d(dst + p * S::PANEL, kv ? &tv : &tk, sm.full + slot, p * (SW / ES), 0, x0.hk, page);
        }
        issued = ld + 1;
      }
      if (!ok) {
        if (lane == 0) *abort_flag = 1;
        break;
      }
      x0 = x1;
      x1 = x2;
    }
    // every slot's latest load lands before the CTA may exit
    for (int ld = max(0, issued - NS); ld < issued; ++ld)
      mbar_wait_w(sm.full + ld % NS, (uint32_t)((ld / NS) & 1), never);
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA issue
    // S(0), S(1), then per tile PV(j) once P(j) is written, and S(j + 2) into the buffer that
    // the softmax of j has read.
    const uint32_t slot_k = (uint32_t)make_smem_desc(smem_u32(base), 16, 8 * SW, LAYOUT);
    const uint32_t q_lo = (uint32_t)make_smem_desc(smem_u32(sQ), 16, 8 * SW, LAYOUT);
    const uint32_t hi_k = (uint32_t)(make_smem_desc(0, 16, 8 * SW, LAYOUT) >> 32);
    // V as the M-major operand: panels of SW bytes of D are LBO apart (a head dim of 64 has one
    // panel, read twice: rows 64-127 of O repeat rows 0-63 and are not used)
    constexpr uint32_t V_LBO = D * ES > SW && ES == 2 ? S::PANEL : 0;
    const uint32_t slot_v = (uint32_t)make_smem_desc(smem_u32(base), V_LBO, 8 * SW, LAYOUT);
    const uint32_t hi_v = (uint32_t)(make_smem_desc(0, V_LBO, 8 * SW, LAYOUT) >> 32);
    // P: 16 bytes of N x 8 positions are contiguous; the next 8 positions are 128 bytes on, the
    // next 16 bytes of N 2048
    const uint32_t p_lo = (uint32_t)make_smem_desc(smem_u32(sP), 128, 2048, SMEM_SWIZZLE_NONE);
    const uint32_t hi_p = (uint32_t)(make_smem_desc(0, 128, 2048, SMEM_SWIZZLE_NONE) >> 32);
    int seg = -1, left_in_seg = 0;
    unsigned starts = 0;  // bit k: the tile k before the one whose S was issued last begins a unit's part
    bool ok = true;
    auto issue_s = [&](int j) -> bool {
      starts <<= 1;
      if (left_in_seg == 0) {
        wk.next(a, &sg);
        left_in_seg = sg.nt;
        ++seg;
        starts |= 1u;
        if (!mbar_wait_w(sm.q_full + (seg & 1), (uint32_t)((seg >> 1) & 1), abort_flag)) return false;
      }
      const int ld = 2 * j, slot = ld % NS;
      if (!mbar_wait_w(sm.full + slot, (uint32_t)((ld / NS) & 1), abort_flag)) return false;
      tc_fence_after();
      const uint32_t ka = slot_k + (uint32_t)((slot * S::SLOT) >> 4), qb = q_lo + (uint32_t)(((seg & 1) * S::QBUF) >> 4);
#pragma unroll
      for (int kk = 0; kk < S::ROWB / 32; ++kk) {
        const uint32_t p = kk * 32 / SW, in = (kk * 32 % SW) >> 4;
        if constexpr (ES == 1)
          mma_f8_ss_w(tmem + (j & 1) * N, ka + p * (S::PANEL >> 4) + in, hi_k, qb + p * (S::QPANEL >> 4) + in, hi_k,
                      IDESC_S, kk > 0);
        else
          mma_ss_w(tmem + (j & 1) * N, ka + p * (S::PANEL >> 4) + in, hi_k, qb + p * (S::QPANEL >> 4) + in, hi_k,
                   IDESC_S, kk > 0);
      }
      tc_commit_w(sm.s_full + (j & 1));
      tc_commit_w(sm.empty + slot);
      if (--left_in_seg == 0) tc_commit_w(sm.q_empty + (seg & 1));
      return true;
    };
    for (int j = 0; j < 2 && ok; ++j) {
      if (j < my_tiles) ok = issue_s(j);
      else starts <<= 1;
    }
    for (int j = 0; j < my_tiles && ok; ++j) {
      const int ld = 2 * j + 1, slot = ld % NS;
      ok = mbar_wait_w(sm.p_full + (j & 1), (uint32_t)((j >> 1) & 1), abort_flag) &&
           mbar_wait_w(sm.full + slot, (uint32_t)((ld / NS) & 1), abort_flag);
      if (!ok) break;
      tc_fence_after();
      const bool fresh = (starts >> 1) & 1u;  // S has been issued one tile beyond j
      const uint32_t pb = p_lo + (uint32_t)(((j & 1) * S::PBUF) >> 4);
#pragma unroll
      for (int db = 0; db < S::NO; ++db) {
        const uint32_t va = slot_v + (uint32_t)((slot * S::SLOT + db * (128 * ES / SW) * S::PANEL) >> 4);
#pragma unroll
        for (int kk = 0; kk < kTile / KPOS; ++kk) {
          const uint32_t acc = (fresh && kk == 0) ? 0u : 1u;
          if constexpr (ES == 1)
            mma_f8_ss_w(tmem + S::TM_O + db * N, va + kk * ((KPOS * SW) >> 4), hi_v, pb + kk * ((KPOS * 16) >> 4),
                        hi_p, IDESC_PV, acc);
          else
            mma_ss_w(tmem + S::TM_O + db * N, va + kk * ((KPOS * SW) >> 4), hi_v, pb + kk * ((KPOS * 16) >> 4), hi_p,
                     IDESC_PV, acc);
        }
      }
      tc_commit_w(sm.empty + slot);
      tc_commit_w(sm.o_full + (j & 1));
      if (j + 2 < my_tiles) ok = issue_s(j + 2);
      else starts <<= 1;
    }
    if (!ok && lane == 0) *abort_flag = 1;
    tc_commit_w(&sm.fin_bar);
    mbar_wait_w(&sm.fin_bar, 0, never);  // every MMA has retired before TMEM is freed
  } else if (warp >= 6) {
    // ---------------------------------------------------------------- Q operand and row constants
    constexpr int TPR = D / 8;          // threads per row, 8 elements each
    constexpr int ROWS = 64 / TPR;      // rows at once
    static_assert(R % ROWS == 0, "whole passes: the shuffles below need full warps");
    const int t = tid - 192, d0 = (t % TPR) * 8;
    bool ok = true;
    for (int seg = 0; ok && wk.next(a, &sg); ++seg) {
      const int buf = seg & 1;
      if (seg >= 2) ok = mbar_wait_w(sm.q_empty + buf, (uint32_t)(((seg >> 1) - 1) & 1), abort_flag);
      if (!ok) break;
      RowConst<R>& rc = sm.rc[buf];
      const bool capped = (a.score.flags & FA_SCORE_SOFTCAP) != 0;
      const float dom = capped ? 1.f : kLog2e;
#pragma unroll 2
      for (int n0 = 0; n0 < R; n0 += ROWS) {
        const int n = n0 + t / TPR;
        const int m = wk.e.rg * R + n, i = m / a.G, h = sg.hk * a.G + (m - i * a.G);
        const bool real = m < a.M, live = real && i < wk.e.ql;
        uint4 raw = make_uint4(0u, 0u, 0u, 0u);
        if (live) {
          const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q.ptr) + (int64_t)wk.e.b * a.q.stride_b +
                               (int64_t)h * a.q.stride_h + (int64_t)i * a.q.stride_t + d0;
          if (a.q_vec) {
            raw = __ldg(reinterpret_cast<const uint4*>(qp));
          } else {
            raw.x = (uint32_t)qp[0] | ((uint32_t)qp[1] << 16);
            raw.y = (uint32_t)qp[2] | ((uint32_t)qp[3] << 16);
            raw.z = (uint32_t)qp[4] | ((uint32_t)qp[5] << 16);
            raw.w = (uint32_t)qp[6] | ((uint32_t)qp[7] << 16);
          }
        }
        float fix = 1.f;  // undoes the row's power of two
        unsigned char* q = sQ + buf * S::QBUF;
        if constexpr (ES == 2) {
          *reinterpret_cast<uint4*>(q + (d0 * 2 / SW) * S::QPANEL + panel_off<SW>(n, (d0 * 2 % SW) >> 4)) = raw;
        } else {
          const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
          float f[8], top = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f[2 * k] = __uint_as_float(w[k] << 16);
            f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
          }
          bool odd = false;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            top = fmaxf(top, fabsf(f[k]));
            odd = odd || !(fabsf(f[k]) < INFINITY);
          }
          if (odd) top = INFINITY;
#pragma unroll
          for (int o = TPR / 2; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          // 2^sh brings the largest magnitude into [128, 256) (at most 2^100: tinier rows stay small)
          const int ex = (int)(__float_as_uint(top) >> 23) - 127;
          const int sh = top > 0.f && top < INFINITY ? min(7 - ex, 100) : 0;
          const float up = __uint_as_float((uint32_t)(sh + 127) << 23);
          fix = __uint_as_float((uint32_t)(127 - sh) << 23);
          if (top == INFINITY) fix = __uint_as_float(0x7fc00000u);  // NaN or infinity in q: the row is NaN
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) hi[k] = split_e4m3x2(f[2 * k] * up, f[2 * k + 1] * up, &lo[k]);
          unsigned char* at = q + (d0 / SW) * S::QPANEL + (d0 & 8);
          const int c = (d0 % SW) >> 4;
          *reinterpret_cast<uint2*>(at + panel_off<SW>(n, c)) = make_uint2(hi[0] | (hi[1] << 16), hi[2] | (hi[3] << 16));
          *reinterpret_cast<uint2*>(at + panel_off<SW>(R + n, c)) =
              make_uint2(lo[0] | (lo[1] << 16), lo[2] | (lo[3] << 16));
        }
        if (d0 == 0) {
          const int qpos = wk.e.len - wk.e.ql + i;
          int lo = 0, hi = wk.e.len - 1;
          if (a.mask.flags & FA_MASK_CAUSAL) hi = min(hi, qpos);
          if (a.mask.flags & FA_MASK_WINDOW) {
            if (a.mask.window_left >= 0) lo = max(lo, qpos - a.mask.window_left);
            if (a.mask.window_right >= 0) hi = (int)min((int64_t)hi, (int64_t)qpos + a.mask.window_right);
          }
          rc.xs[n] = a.scale * fix * dom;
          rc.slope[n] = live && (a.score.flags & FA_SCORE_ALIBI) ? __ldg(a.score.alibi_slopes + h) * dom : 0.f;
          rc.lo[n] = live ? lo : 1;
          rc.hi[n] = live ? hi : 0;
          rc.qpos[n] = qpos;
          rc.orow[n] = real ? (int64_t)wk.e.b * a.o.stride_b + (int64_t)h * a.o.stride_h + (int64_t)i * a.o.stride_t : -1;
          rc.lrow[n] = ((int64_t)wk.e.b * a.H + h) * a.Tq + i;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.q_full + buf);
    }
    // Entries without a tile: their rows see nothing.
    const int t64 = tid - 192;
    for (int e = cta; e < a.entries; e += gridDim.x) {
      const Entry x = entry_of<R>(a, e);
      if (x.nt) continue;
      const int m0 = x.rg * R, rows = min(R, a.M - m0);
      for (int k = t64; k < a.Hkv * rows * D; k += 64) {
        const int d = k % D, r = k / D, hk = r / rows, m = m0 + r % rows, i = m / a.G, h = hk * a.G + m % a.G;
        reinterpret_cast<uint16_t*>(a.o.ptr)[(int64_t)x.b * a.o.stride_b + (int64_t)h * a.o.stride_h +
                                             (int64_t)i * a.o.stride_t + d] = 0;
        if (d == 0) a.lse[((int64_t)x.b * a.H + h) * a.Tq + i] = -INFINITY;
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax (thread = position)
    RowState<R>& rs = sm.rs;
    const uint32_t t_lane = tmem + ((uint32_t)(warp * 32) << 16);
    const bool capped = (a.score.flags & FA_SCORE_SOFTCAP) != 0, alibi = (a.score.flags & FA_SCORE_ALIBI) != 0;
    const float cap2 = capped ? a.score.softcap * kLog2e : 0.f, cap_k = capped ? 2.f * kLog2e / a.score.softcap : 0.f;
    constexpr int RC = R < 32 ? R : 32;        // rows per TMEM read (x2 parts for 8-bit codes)
    constexpr int PW = 16 / ES;                // columns per 16-byte store of P
    int unit0 = -1, unit1 = -1, j = 0;
    for (int seg = 0; wk.next(a, &sg); ++seg) {
      const RowConst<R>& rc = sm.rc[seg & 1];
      if (tid < R) {
        rs.mx[tid] = rs.my[tid] = rs.thx[tid] = rs.thy[tid] = -INFINITY;
        rs.mref[tid] = 0.f;
        rs.w[tid] = 1.f;
      }
      if (!mbar_wait(sm.q_full + (seg & 1), (uint32_t)((seg >> 1) & 1), abort_flag)) *abort_flag = 1;
      named_bar_sync(1, 128);
      float l[R];
#pragma unroll
      for (int n = 0; n < R; ++n) l[n] = 0.f;
      for (int it = 0; it < sg.nt; ++it, ++j) {
        const int pos = (sg.t0 + it) * kTile + tid;
        // No wait leaves the loop: after a time-out every later wait returns at once and nothing
        // is written at the end.
        if (!mbar_wait(sm.s_full + (j & 1), (uint32_t)((j >> 1) & 1), abort_flag)) *abort_flag = 1;
        tc_fence_after();
        const float2 sc = sm.scales[j % kScaleRing][tid / a.ps];
        const bool shown = sc.x != -INFINITY;
        const float ks = shown ? sc.x : 0.f, vs = sc.y;
        const int p0 = (sg.t0 + it) * kTile;
        const bool inside = p0 >= wk.e.in_lo && p0 + kTile - 1 <= wk.e.in_hi && !sm.odd[j % kScaleRing];
        // a scale below 2^-100 (none that an append makes) counts as 2^-100 here: w stays finite
        const float lv = ES == 1 ? fmaxf(lg2_approx(vs), -100.f) : 0.f;
        float x[R];
        bool over = false;
#pragma unroll
        for (int c = 0; c < R; c += RC) {
          if constexpr (ES == 1) {
            constexpr int W = R == 8 ? 16 : RC;  // R = 8: hi and lo parts in one read
            uint32_t h[W], lo[W];
            tmem_cols<W>(t_lane + (j & 1) * N + c, h);
            if constexpr (R > 8) tmem_cols<W>(t_lane + (j & 1) * N + R + c, lo);
            tmem_ld_wait();
            reg_pin(h);
            if constexpr (R > 8) reg_pin(lo);
#pragma unroll
            for (int n = 0; n < RC; ++n)
              x[c + n] = fmaf(__uint_as_float(R == 8 ? h[(8 + n) % W] : lo[n]), 0.0625f, __uint_as_float(h[n]));
          } else {
            uint32_t h[RC];
            tmem_cols<RC>(t_lane + (j & 1) * N + c, h);
            tmem_ld_wait();
            reg_pin(h);
#pragma unroll
            for (int n = 0; n < RC; ++n) x[c + n] = __uint_as_float(h[n]);
          }
        }
#pragma unroll
        for (int n = 0; n < R; ++n) x[n] *= ES == 1 ? ks * rc.xs[n] : rc.xs[n];
        if (alibi) {
#pragma unroll
          for (int n = 0; n < R; ++n) x[n] = fmaf(rc.slope[n], (float)(pos - rc.qpos[n]), x[n]);
        }
        if (capped) {  // cap tanh(x / cap) = cap (1 - 2 / (1 + e^(2 x / cap))), in log2 units
#pragma unroll
          for (int n = 0; n < R; ++n) x[n] = fmaf(-2.f * cap2, __fdividef(1.f, 1.f + ex2_approx(x[n] * cap_k)), cap2);
        }
        if (!inside) {
#pragma unroll
          for (int n = 0; n < R; ++n)
            if (!shown || pos < rc.lo[n] || pos > rc.hi[n]) x[n] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < R; ++n) over = over || x[n] > (ES == 1 ? fminf(rs.thx[n], rs.thy[n] - lv) : rs.thx[n]);
        if (vote_or(1, 128, over)) {
          // ---- a reference has to move: the tile's largest x (and x + lv) per row
#pragma unroll
          for (int n = 0; n < R; ++n) {
            const float mx = warp_max(x[n]), my = ES == 1 ? warp_max(x[n] + lv) : 0.f;
            if (lane == (n & 31)) {
              rs.red[warp][0][n] = mx;
              if (ES == 1) rs.red[warp][1][n] = my;
            }
          }
          named_bar_sync(1, 128);
          if (tid < R) {
            const int n = tid;
            const float ox = rs.mx[n], oy = rs.my[n];
            const float nx = fmaxf(fmaxf(rs.red[0][0][n], rs.red[1][0][n]), fmaxf(rs.red[2][0][n], rs.red[3][0][n]));
            const float mx = nx > ox + kSlack ? nx : ox;
            float my = mx;
            if constexpr (ES == 1) {
              const float ny = fmaxf(fmaxf(rs.red[0][1][n], rs.red[1][1][n]), fmaxf(rs.red[2][1][n], rs.red[3][1][n]));
              my = ny > oy + kSlack ? ny : oy;
            }
            rs.al[n] = mx != ox ? ex2_approx(ox - mx) : 1.f;
            rs.ao[n] = my != oy ? ex2_approx(oy - my) : 1.f;
            const float mref = mx == -INFINITY ? 0.f : mx;
            rs.mx[n] = mx;
            rs.my[n] = my;
            rs.mref[n] = mref;
            rs.thx[n] = mx + kSlack;
            rs.thy[n] = my + kSlack;
            rs.w[n] = ES == 1 && my != -INFINITY ? ex2_approx(mref - my + kLift) : 1.f;
          }
          named_bar_sync(1, 128);
#pragma unroll
          for (int n = 0; n < R; ++n) l[n] *= rs.al[n];
          if (it > 0) {  // O holds earlier tiles' sums: PV(j - 1) must have retired
            if (!mbar_wait(sm.o_full + ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag)) *abort_flag = 1;
            tc_fence_after();
            constexpr int W = N < 32 ? N : 32;
#pragma unroll 1
            for (int c = 0; c < S::NO * N; c += W) {
              uint32_t o[W];
              tmem_cols<W>(t_lane + S::TM_O + c, o);
              tmem_ld_wait();
              reg_pin(o);
#pragma unroll
              for (int k = 0; k < W; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * rs.ao[(c + k) % R]);
              tmem_put<W>(t_lane + S::TM_O + c, o);
            }
            tmem_st_wait();
          }
        }
        // ---- probabilities: the sum in fp32, P into shared memory as the B operand
        if (j >= 2 && !mbar_wait(sm.o_full + (j & 1), (uint32_t)(((j >> 1) - 1) & 1), abort_flag)) *abort_flag = 1;
        unsigned char* pw = sP + (j & 1) * S::PBUF + (tid >> 3) * 128 + (tid & 7) * 16;
#pragma unroll
        for (int n = 0; n < R; ++n) {
          const float p = ex2_approx(x[n] - rs.mref[n]);
          l[n] += p;
          x[n] = ES == 1 ? p * (rs.w[n] * vs) : p;
        }
        if constexpr (ES == 2) {
#pragma unroll
          for (int g = 0; g < R / PW; ++g) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = pack_bf16x2(x[g * PW + 2 * k], x[g * PW + 2 * k + 1]);
            *reinterpret_cast<uint4*>(pw + g * 2048) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        } else {
          uint32_t hi[R / 4], lo[R / 4];
#pragma unroll
          for (int k = 0; k < R / 4; ++k) {
            uint32_t l0, l1;
            const uint32_t h0 = split_e4m3x2(x[4 * k], x[4 * k + 1], &l0);
            const uint32_t h1 = split_e4m3x2(x[4 * k + 2], x[4 * k + 3], &l1);
            hi[k] = h0 | (h1 << 16);
            lo[k] = l0 | (l1 << 16);
          }
          if constexpr (R == 8) {
            *reinterpret_cast<uint4*>(pw) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
          } else {
#pragma unroll
            for (int g = 0; g < R / 16; ++g) {
              *reinterpret_cast<uint4*>(pw + g * 2048) = make_uint4(hi[4 * g], hi[4 * g + 1], hi[4 * g + 2], hi[4 * g + 3]);
              *reinterpret_cast<uint4*>(pw + (R / 16 + g) * 2048) =
                  make_uint4(lo[4 * g], lo[4 * g + 1], lo[4 * g + 2], lo[4 * g + 3]);
            }
          }
        }
        if (p0 < wk.e.lo || p0 + kTile - 1 > wk.e.hi) {
          // Positions that no row sees may hold anything (a zero probability times NaN is NaN):
          // their rows of V become zero once the tile has landed.
          const int ld = 2 * j + 1, slot = ld % NS;
          if (!mbar_wait(sm.full + slot, (uint32_t)((ld / NS) & 1), abort_flag)) *abort_flag = 1;
          if (pos < wk.e.lo || pos > wk.e.hi) {
            unsigned char* v = base + (size_t)slot * S::SLOT + tid * SW;
#pragma unroll
            for (int p = 0; p < S::ROWB / SW; ++p)
#pragma unroll
              for (int c = 0; c < SW / 16; ++c)
                *reinterpret_cast<uint4*>(v + p * S::PANEL + c * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(sm.p_full + (j & 1));
      }
      // ---- end of the unit's part: join the threads' sums, scale O and write it
#pragma unroll
      for (int n = 0; n < R; ++n) {
        float v = l[n];
#pragma unroll
        for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == (n & 31)) rs.red[warp][0][n] = v;
      }
      named_bar_sync(1, 128);
      if (!mbar_wait(sm.o_full + ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1), abort_flag)) *abort_flag = 1;
      tc_fence_after();
      const bool whole = sg.first && sg.last;
      const int part = 2 * cta + (seg == 0 ? 0 : 1);
      const int unit = 2 * (wk.idx * a.Hkv + sg.hk) + (sg.first ? 1 : 0);
      const bool good = !*abort_flag;
      if (!whole) (seg == 0 ? unit0 : unit1) = unit;
      if (tid < R) {
        const int n = tid;
        const float sum = (rs.red[0][0][n] + rs.red[1][0][n]) + (rs.red[2][0][n] + rs.red[3][0][n]);
        // a NaN stays one; a row that may see nothing took part in the tiles that needed no mask
        const bool some = !(sum == 0.f) && rc.lo[n] <= rc.hi[n];
        rs.fin[n] = some ? 1.f / (rs.w[n] * sum) : 0.f;
        const float lse = some ? (rs.mref[n] + log2f(sum)) * kLn2 : -INFINITY;
        if (good) {
          if (!whole) a.part_lse[(int64_t)part * R + n] = lse;
          else if (rc.orow[n] >= 0) a.lse[rc.lrow[n]] = lse;
        }
      }
      named_bar_sync(1, 128);
      if (D >= 128 || warp < 2) {
        constexpr int W = R < 16 ? 16 : (R < 32 ? 16 : 32);  // columns per read
#pragma unroll 1
        for (int db = 0; db < S::NO; ++db) {
          const int d = db * 128 + tid;
#pragma unroll 1
          for (int c = 0; c < R; c += W) {
            const uint32_t at = t_lane + S::TM_O + db * N + c;
            uint32_t h[W], lo[W];
            tmem_cols<W>(at, h);
            if constexpr (ES == 1 && R > 8) tmem_cols<W>(at + R, lo);
            tmem_ld_wait();
            reg_pin(h);
            if constexpr (ES == 1 && R > 8) reg_pin(lo);
#pragma unroll
            for (int k = 0; k < (R < W ? R : W); ++k) {
              float v = __uint_as_float(h[k]);
              if constexpr (ES == 1) v = fmaf(__uint_as_float(R == 8 ? h[(8 + k) % W] : lo[k]), 0.0625f, v);
              v *= rs.fin[c + k];
              if (!good) continue;
              if (!whole) {
                a.part_o[((int64_t)part * R + c + k) * D + d] = v;
              } else if (rc.orow[c + k] >= 0) {
                reinterpret_cast<__nv_bfloat16*>(a.o.ptr)[rc.orow[c + k] + d] = __float2bfloat16_rn(v);
              }
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(sm.q_empty + (seg & 1));
    }
    if (tid == 0) {
      a.part_unit[2 * cta] = unit0;
      a.part_unit[2 * cta + 1] = unit1;
      if (*abort_flag) report_status(a.status, FA_ERR_TIMEOUT);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TM_COLS);
  }
}

// Joins the parts of the unit that begins in CTA blockIdx.x and runs on into the next ones, in CTA
// order: one warp per query row.  Launched with programmatic serialisation, so that its blocks are
// resident when the last CTA of the attention kernel ends.
template <int D, int R>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedArgs a, const int ctas) {
  __shared__ float w_sh[8][2 * kSms + 2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x, n = blockIdx.y * 8 + warp;
  griddep_wait();
  const int u0 = a.part_unit[2 * c], u1 = a.part_unit[2 * c + 1];
  int first, key;
  if (u1 >= 0) {
    first = 2 * c + 1;
    key = u1 >> 1;
  } else if (u0 >= 0 && (u0 & 1)) {
    first = 2 * c;
    key = u0 >> 1;
  } else {
    return;
  }
  int parts = 1;  // the unit's parts: `first`, then slot 2 (c + k) of the CTAs that follow
  for (int k = c + 1; k < ctas; k += 32) {
    const bool same = k + lane < ctas && a.part_unit[2 * (k + lane)] == 2 * key;
    const unsigned m = __ballot_sync(0xffffffffu, same);
    const int run = m == 0xffffffffu ? 32 : __ffs(~m) - 1;
    parts += run;
    if (run < 32) break;
  }
  const int e = key / a.Hkv, hk = key % a.Hkv, b = e / a.groups, m = (e % a.groups) * R + n;
  if (n >= R || m >= a.M) return;
  auto slot = [&](int k) -> int64_t { return k == 0 ? first : 2 * (c + k); };
  float* w = w_sh[warp];
  float top = -INFINITY;
  for (int k = lane; k < parts; k += 32) top = fmaxf(top, a.part_lse[slot(k) * R + n]);
  top = warp_max(top);
  const float ref = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int k = lane; k < parts; k += 32) {
    const float v = expf(a.part_lse[slot(k) * R + n] - ref);
    w[k] = v;
    sum += v;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncwarp();
  float acc[D / 32];
#pragma unroll
  for (int k = 0; k < D / 32; ++k) acc[k] = 0.f;
#pragma unroll 4
  for (int k = 0; k < parts; ++k) {
    const float* po = a.part_o + (slot(k) * R + n) * D + lane;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(w[k], po[32 * i], acc[i]);
  }
  const int i = m / a.G, h = hk * a.G + m % a.G;
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.o.ptr) + (int64_t)b * a.o.stride_b +
                     (int64_t)h * a.o.stride_h + (int64_t)i * a.o.stride_t;
  const bool some = !(sum == 0.f);
  const float inv = some ? 1.f / sum : 0.f;
#pragma unroll
  for (int k = 0; k < D / 32; ++k) o[lane + 32 * k] = __float2bfloat16_rn(acc[k] * inv);
  if (lane == 0) a.lse[((int64_t)b * a.H + h) * a.Tq + i] = some ? ref + logf(sum) : -INFINITY;
}

struct PagedPlan {
  int R, groups, ctas;
  size_t workspace;
};

// Rows per group: the smallest operand width that holds every query row of a K/V head, or 64
// (32 for bf16 pages of head dim 256, whose tiles leave no room for more) with as many groups as
// it takes, each reading the cache again.
PagedPlan plan_paged(const FaPagedAttnParams* p) {
  PagedPlan pl;
  const bool f8 = p->cache.dtype == FA_DTYPE_E4M3;
  const int64_t M = (int64_t)(p->H / p->cache.H_kv) * p->Tq;
  const int top = !f8 && p->cache.D == 256 ? 32 : 64;
  pl.R = f8 ? 8 : 16;
  while (pl.R < M && pl.R < top) pl.R *= 2;
  pl.groups = (int)((M + pl.R - 1) / pl.R);
  const int64_t tiles = (int64_t)p->B * pl.groups * p->cache.H_kv *
                        (((int64_t)p->cache.table_cols * p->cache.page_size + kTile - 1) / kTile);
  pl.ctas = (int)std::min<int64_t>(kSms, tiles);
  pl.workspace = (size_t)2 * pl.ctas * ((size_t)pl.R * (p->cache.D + 1) * 4 + 4) + 256;
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

template <int D, int ES, int R>
cudaError_t launch_paged(const CUtensorMap& tk, const CUtensorMap& tv, PagedArgs& a, const PagedPlan& pl,
                         cudaStream_t stream) {
  const size_t fixed = paged_smem_bytes<D, ES, R>(0), limit = 232448;
  a.slots = (int)std::min<size_t>(kMaxSlots, (limit - fixed) / Shape<D, ES, R>::SLOT);
  const size_t smem = paged_smem_bytes<D, ES, R>(a.slots);
  cudaError_t e =
      cudaFuncSetAttribute(paged_attn_kernel<D, ES, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  paged_attn_kernel<D, ES, R><<<pl.ctas, kPThreads, smem, stream>>>(tk, tv, a);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  if (a.cols * a.ps <= kTile) return cudaSuccess;  // one tile per unit: no unit crosses CTAs
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)pl.ctas, (unsigned)((R + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_merge_kernel<D, R>, (const PagedArgs)a, (int)pl.ctas);
}

template <int D>
cudaError_t launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, PagedArgs& a, const PagedPlan& pl, bool f8,
                        cudaStream_t st) {
  if (f8) {
    switch (pl.R) {
      case 8: return launch_paged<D, 1, 8>(tk, tv, a, pl, st);
      case 16: return launch_paged<D, 1, 16>(tk, tv, a, pl, st);
      case 32: return launch_paged<D, 1, 32>(tk, tv, a, pl, st);
      default: return launch_paged<D, 1, 64>(tk, tv, a, pl, st);
    }
  }
  if (pl.R == 16) return launch_paged<D, 2, 16>(tk, tv, a, pl, st);
  if (D == 256 || pl.R == 32) return launch_paged<D, 2, 32>(tk, tv, a, pl, st);
  if constexpr (D < 256) return launch_paged<D, 2, 64>(tk, tv, a, pl, st);
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
  a.ps = c.page_size;
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
  a.part_unit = reinterpret_cast<int32_t*>(a.part_lse + (size_t)2 * pl.ctas * pl.R);
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
