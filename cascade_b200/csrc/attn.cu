// Attention over KV caches: causal prompts and trees of drafted tokens, with
// grouped heads, over cached tokens in pages followed by new packed tokens.
#include <cfloat>
#include <type_traits>

#include "attn.cuh"
#include "kernels.cuh"

namespace cb {
namespace attn {
namespace {

constexpr int kThreads = 512;    // 2 softmax warpgroups, 4 loaders, 4 for MMAs
constexpr int kMaxSlots = 12;

struct FwdArgs {
  KvSource kv;
  const char *q;
  int64_t q_tok, q_head;           // bytes
  char *out;
  int64_t o_tok, o_head;           // bytes
  float *lse;
  int64_t l_tok, l_head;           // elements
  const uint8_t *mask;
  int64_t mask_row;
  const int32_t *plan;
  float *part_o, *part_lse;        // [slot][row tile rows][D], [slot][rows]
  int ctas, group, tree, give_up;
  int out32;                       // rows of out are 32-byte aligned
  float scale, c;                  // c = scale * log2(e)
};

// Shared memory: the Q tile(s), a ring of K and V tiles, then this.
struct Control {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t q_full, q_empty;
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t turn[2];
  uint64_t done;
  alignas(16) uint32_t valid[8][4];  // which keys of a tile there are
  float2 ml[2][kTile];             // two key tiles: each chain's (max, sum)
  uint32_t tmem, sent[4];          // the latter: items of each loader warp
  int give_up;
  int bad_v;                       // a masked tile held inf or NaN
};

// Three forms of the kernel, by the rows of an item.
enum Form {
  kTwoRows,      // up to 256: two row tiles take turns on each key tile
  kTwoKeys,      // up to 128: one row tile, two key tiles at a time
  kFewRows,      // up to 16: the same, and the four warps of a warpgroup
};               // share out a key tile's columns

template <int D, int kForm>
struct Shape {
  static constexpr bool kDual = kForm != kTwoRows;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kQTiles = kDual ? 1 : 2;
  // the form for few rows joins its warps' results in one tile's room
  static constexpr int kJoin = kForm == kFewRows ? 1 : 0;
  static constexpr int kSlots =
      D == 128 ? (kDual ? 6 - kJoin : 5) : 12 - kJoin;
  static constexpr int kAhead = kDual ? 2 : 1;
  static constexpr int kSmem =
      (kQTiles + kSlots + kJoin) * kTileBytes + (int)sizeof(Control);
  static_assert(kSlots <= kMaxSlots, "ring");
  static_assert(kSmem <= 232448, "shared memory of one SM");
};

// The lse of a part whose row saw keys, all of scores of -inf.
constexpr float kNoWeight = -FLT_MAX;

// First key tile of an item in which some row does not see every key.
__device__ __forceinline__ int first_masked_tile(const Segment &s, int group,
                                                 int tree) {
  return (s.cached + (tree ? 0 : s.row0 / group + 1)) / kTile;
}

// A row's maximum grows to m_new: its sum and its row of O follow.
template <int D>
__device__ __forceinline__ void raise_maximum(float &m, float &l, float m_new,
                                              bool first, float c,
                                              uint32_t tm_o) {
  if (!first) {
    const float f = m == -INFINITY ? (l == 0.f ? 1.f : 0.f)
                                   : ex2((m - m_new) * c);
    l *= f;
#pragma unroll 1
    for (int i = 0; i < D / 16; ++i) {
      uint32_t o[16];
      tc_ld16(o, tm_o + i * 16);
      tc_wait_ld();
      tc_hold(o);
#pragma unroll
      for (int e = 0; e < 16; ++e)
        o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
      tc_st16(tm_o + i * 16, o);
    }
  }
  m = m_new;
}

// The part of one value of O that zeros stood in for: a row of V that a
// masked tile had cleared of inf and NaN gives them back to rows that see it.
template <bool kBf16>
__device__ __forceinline__ float cleared(uint16_t bits) {
  constexpr uint16_t ex = kBf16 ? 0x7f80 : 0x7c00;
  constexpr uint16_t mant = kBf16 ? 0x007f : 0x03ff;
  if ((bits & ex) != ex) return 0.f;
  return (bits & mant) ? NAN : (bits & 0x8000) ? -INFINITY : INFINITY;
}

// Adds those of the segment's masked tiles [from, to) to kN columns.
template <bool kBf16, int kN>
__device__ __forceinline__ void give_back(float (&o)[kN], const KvSource &kv,
                                          const Segment &sg, int from, int to,
                                          int lim, const uint8_t *mrow,
                                          int col) {
  const int end = min(to * kTile, sg.cached + sg.n_new);
  for (int j = from * kTile; j < end; ++j) {
    const char *vp;
    if (j < sg.cached) {
      const int id = page_of(kv, sg.b, j);
      if (id < 0) continue;
      vp = kv.vp + id * kv.vp_page + sg.hk * kv.vp_head +
           (j % kv.page) * kv.vp_tok;
    } else {
      if (mrow != nullptr ? !mrow[j - sg.cached] : j >= lim) continue;
      vp = kv.v + (int64_t)(sg.tok0 + j - sg.cached) * kv.v_tok +
           sg.hk * kv.v_head;
    }
#pragma unroll
    for (int e = 0; e < kN; ++e)
      o[e] += cleared<kBf16>(reinterpret_cast<const uint16_t *>(vp)[col + e]);
  }
}

// ------------------------------------------------------------------ kernel
// Mathematics.  Row r of an item is (token i, head g of the group): s_rj =
// scale q_r . k_j over the visible keys j, o_r = sum_j softmax_j(s_rj) v_j,
// in one pass over the key tiles with a running maximum m and sum l per row.
// The heads of a group are rows of one item, so K and V are read once per
// group.  S = Q K^T and O += P V run on tcgen05 with 128-row tiles: S, P and
// O stay in TMEM, P (rounded to the inputs' 16 bits, as an MMA operand must
// be; its sum l is taken in FP32 before the rounding) overwrites its own S,
// and a thread owns one row, so no reduction crosses threads.  O is rescaled
// only when a row's maximum grew by more than 2^8, so weights reach 2^8; in
// FP16 they are scaled by 2^7 besides, to 2^15 at most (its largest is 2^16),
// so that weights down to 2^-21 of the largest keep all their bits.
//
// Roles.  Two softmax warpgroups, four loader warps that keep a ring of K and
// V tiles full (TMA for whole tiles, cp.async for ragged ones), and one or two
// warps that issue MMAs; mbarriers between them.  Three forms, by rows:
// - more than 128: two row tiles share each K and V tile and take turns (one's
//   MMAs run under the other's exponentials);
// - up to 128: one row tile, and the warpgroups take alternate key tiles, each
//   with its own m, l and O, joined in the epilogue;
// - up to 16 (decode): as the last, and Q's rows are there four times, one for
//   each warp of a warpgroup, which takes 32 of a tile's 128 keys.
//
// What bounds it (B200, D = 128).  Prompts: the chain of a row tile, softmax
// (about 2100 cycles a tile, of which 1024 on the special-function unit) then
// PV and QK (1040 cycles of MMA and 300 of hand-over), two chains at a time:
// 16384 tokens of 64 heads take 3.8 ms in a run of ten calls, 1160 TFLOP/s, and
// 4.3 to 4.4 ms, 1010 TFLOP/s, in a long run under the power cap.  Decode: HBM;
// 64 sequences of 4200 tokens read 1.12 GB in 179 us a call on one cache over
// and over, 6.2 TB/s, and in 198 to 214 us on caches that change.
template <int D, bool kBf16, int kForm>
__global__ void __launch_bounds__(kThreads, 1)
    attn_fwd_kernel(const __grid_constant__ FwdArgs a,
                    const __grid_constant__ TileMaps maps) {
  using Sh = Shape<D, kForm>;
  constexpr bool kDual = Sh::kDual, kFew = kForm == kFewRows;
  // P and l are 2^kShift times the weights, so that fewer of them fall below
  // 2^-14, where FP16 has fewer bits
  constexpr float kShift = kBf16 ? 0.f : 7.f;
  constexpr float kUnshift = kBf16 ? 1.f : 0x1p-7f;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sm_q = smem_u32(smem);
  const uint32_t sm_ring = sm_q + Sh::kQTiles * Sh::kTileBytes;
  Control &ct = *reinterpret_cast<Control *>(
      smem + (Sh::kQTiles + Sh::kSlots + Sh::kJoin) * Sh::kTileBytes);
  volatile int *give_up = &ct.give_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (sm_q & 1023) {               // the swizzle needs 1024-byte alignment
    if (threadIdx.x == 0) atomicAdd(&g_timeouts, 1u);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < Sh::kSlots; ++i) {
      mbar_init(smem_u32(&ct.full[i]), 128 + 4);
      mbar_init(smem_u32(&ct.empty[i]), kDual ? 1 : 2);
    }
    mbar_init(smem_u32(&ct.q_full), 128 + 4);
    mbar_init(smem_u32(&ct.q_empty), kDual ? 1 : 2);
    mbar_init(smem_u32(&ct.done), kDual ? 1 : 2);
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&ct.s_full[w]), 1);
      mbar_init(smem_u32(&ct.p_full[w]), 4);
      mbar_init(smem_u32(&ct.o_full[w]), 1);
      mbar_init(smem_u32(&ct.turn[w]), 1);
    }
    ct.give_up = a.give_up;
    if (a.give_up) atomicAdd(&g_timeouts, 1u);
    ct.bad_v = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // The launch may be early: what is in memory may be what the kernel before
  // this one writes, the plan included.  TMEM too is taken behind the wait:
  // a block of that kernel that shares the SM may still have to get its own,
  // and each would wait for the other.  The next kernel may start once it is
  // taken.
  wait_for_previous();
  if (warp == 12) tc_alloc(smem_u32(&ct.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  const uint32_t tmem = ct.tmem;
  const Segment *segs =
      reinterpret_cast<const Segment *>(a.plan + seg_offset(a.ctas));
  const int seg_begin = a.plan[blockIdx.x], seg_end = a.plan[blockIdx.x + 1];

  if (warp < 8) {
    // ------------------------------------------------------ softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int w = warp >> 2;                       // warpgroup
    const int rt = (warp & 3) * 32 + lane;         // row of the tile
    // row of the item: in the form for few rows every warp has them all
    const int r = kFew ? lane : (kDual ? 0 : w * kTile) + rt;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t tm_s = lane_base + w * 128;
    const uint32_t tm_o = lane_base + 256 + w * 128;
    const float grow = 8.f / a.c;                  // allowed growth of m
    uint32_t s_phase = 0, o_phase = 0, o_phase2 = 0;
    int tiles_done = 0;
    bool on = true;                      // no wait was let through
    for (int si = seg_begin; si < seg_end; ++si) {
      const Segment sg = segs[si];
      const int n_end = kDual ? sg.t1 : (w ? sg.n1 : sg.n0);
      const int t_all = kDual ? sg.t1 : max(sg.n0, sg.n1);
      const int t_first = kDual ? sg.t0 + w : sg.t0;
      const bool warp_on = r - lane < sg.rows;
      const bool row_on = r < sg.rows;
      const int tok = (sg.row0 + r) / a.group;
      const int head = sg.hk * a.group + (sg.row0 + r) - tok * a.group;
      // causal: keys below lim are visible; tree: cached ones and the mask's
      const int lim =
          !row_on ? 0 : a.tree ? sg.cached : sg.cached + tok + 1;
      const int masked_from = first_masked_tile(sg, a.group, a.tree);
      const uint8_t *mrow =
          a.tree && row_on ? a.mask + (int64_t)(sg.tok0 + tok) * a.mask_row
                           : nullptr;
      float m = -INFINITY, l = 0.f;
      bool seen = false, first = true;
      for (int t = t_first; t < n_end; t += kDual ? 2 : 1) {
        on = mbar_wait(smem_u32(&ct.s_full[w]), s_phase, give_up) && on;
        s_phase ^= 1;
        if constexpr (kFew) {
          // This warp's 32 of the tile's 128 keys.  Its rows of P are zero
          // at the other warps' keys, so its rows of O are the part of its
          // own: eight parts of each row are joined in the epilogue.
          const int part = warp & 3;
          tc_fence_after();
          uint32_t x[32];
          tc_ld32(x, tm_s + part * 32);
          uint32_t vis = ct.valid[(tiles_done + t - sg.t0) & 7][part];
          if (t >= masked_from) {
            const int j0 = t * kTile + part * 32;
            const int nvis = min(max(lim - j0, 0), 32);
            uint32_t own = nvis == 32 ? 0xffffffffu : (1u << nvis) - 1;
            if (mrow != nullptr && j0 + 32 > sg.cached) {
              const int e = min(j0 + 32, sg.cached + sg.n_new);
              for (int j = max(j0, sg.cached); j < e; ++j)
                if (mrow[j - sg.cached]) own |= 1u << (j - j0);
            }
            vis &= own;
          }
          seen |= vis != 0;
          tc_wait_ld();
          tc_hold(x);
          if (!__all_sync(0xffffffffu, vis == 0xffffffffu)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!((vis >> e) & 1)) x[e] = 0xff800000u;    // -inf
          }
          float t0 = __uint_as_float(x[0]), t1 = __uint_as_float(x[1]);
#pragma unroll
          for (int e = 2; e < 32; e += 2) {
            t0 = fmaxf(t0, __uint_as_float(x[e]));
            t1 = fmaxf(t1, __uint_as_float(x[e + 1]));
          }
          const float top = fmaxf(t0, t1);
          if (__any_sync(0xffffffffu, top > m + grow))
            raise_maximum<D>(m, l, fmaxf(m, top), first, a.c, tm_o);
          first = false;
          const float mc = m == -INFINITY ? 0.f : fmaf(m, a.c, -kShift);
          const uint64_t c2 = pair_of(a.c, a.c), m2 = pair_of(-mc, -mc);
          uint64_t sum[2] = {0, 0};
          uint32_t p[16], none[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            p[e] = weigh2<kBf16>(x[2 * e], x[2 * e + 1], c2, m2, sum[e & 1]);
            none[e] = 0;
          }
          float s0, s1;
          unpair(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i == part)
              tc_st16(tm_s + i * 16, p);
            else
              tc_st16(tm_s + i * 16, none);
          tc_wait_st();
          tc_fence_before();
        } else if (warp_on) {
          tc_fence_after();
          uint32_t x[4][32];
#pragma unroll
          for (int i = 0; i < 4; ++i) tc_ld32(x[i], tm_s + i * 32);
          const uint32_t *there = ct.valid[(tiles_done + t - sg.t0) & 7];
          const uint4 vw = *reinterpret_cast<const uint4 *>(there);
          if ((vw.x & vw.y & vw.z & vw.w) != 0xffffffffu || t >= masked_from) {
            // What a row does not see becomes -inf in TMEM, 32 keys at a
            // time: a loop, because unrolled its code would push the hot
            // loops out of the instruction cache.
            tc_wait_ld();
            uint32_t any = 0;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
              const int j0 = t * kTile + i * 32;
              const int nvis = min(max(lim - j0, 0), 32);
              uint32_t vis = nvis == 32 ? 0xffffffffu : (1u << nvis) - 1;
              if (mrow != nullptr && j0 + 32 > sg.cached) {
                const int e = min(j0 + 32, sg.cached + sg.n_new);
                for (int j = max(j0, sg.cached); j < e; ++j)
                  if (mrow[j - sg.cached]) vis |= 1u << (j - j0);
              }
              vis &= there[i];
              any |= vis;
              // most 32-key pieces of a masked tile are seen whole
              if (__all_sync(0xffffffffu, vis == 0xffffffffu)) continue;
              uint32_t z[32];
              tc_ld32(z, tm_s + i * 32);
              tc_wait_ld();
              tc_hold(z);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!((vis >> e) & 1)) z[e] = 0xff800000u;
              tc_st32(tm_s + i * 32, z);
            }
            tc_wait_st();
            seen |= any != 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) tc_ld32(x[i], tm_s + i * 32);
          } else {
            seen = true;
          }
          tc_wait_ld();
#pragma unroll
          for (int i = 0; i < 4; ++i) tc_hold(x[i]);
          float mx[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            mx[i] = fmaxf(__uint_as_float(x[i][0]), __uint_as_float(x[i][1]));
#pragma unroll
            for (int e = 2; e < 32; ++e)
              mx[i] = fmaxf(mx[i], __uint_as_float(x[i][e]));
          }
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
          // m == -inf: any finite top is growth
          if (__any_sync(0xffffffffu, top > m + grow))
            raise_maximum<D>(m, l, fmaxf(m, top), first, a.c, tm_o);
          first = false;
          const float mc = m == -INFINITY ? 0.f : fmaf(m, a.c, -kShift);
          const uint64_t c2 = pair_of(a.c, a.c), m2 = pair_of(-mc, -mc);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t p[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              p[e] = weigh2<kBf16>(x[i][2 * e], x[i][2 * e + 1], c2, m2,
                                   sum[e & 1]);
            tc_st16(tm_s + i * 16, p);
          }
          float s0, s1;
          unpair(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
          tc_wait_st();
          tc_fence_before();
        }
        __syncwarp();
        if (lane == 0 && on) mbar_arrive(smem_u32(&ct.p_full[w]));
      }
      tiles_done += t_all - sg.t0;

      // ---------------------------------------------------- epilogue
      if constexpr (kFew) {
        const int part = warp & 3;
        const bool steps = n_end > t_first;
        const bool steps2 = w ? true : sg.t1 > sg.t0 + 1;
        ct.ml[w][rt] = make_float2(m, seen && l == 0.f ? -1.f : l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        float mm = -INFINITY, lsum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          mm = fmaxf(mm, ct.ml[i >> 2][(i & 3) * 32 + lane].x);
        const float mc = mm == -INFINITY ? 0.f : mm * a.c;
        float f1 = 0.f, f2 = 0.f;          // factors of this warp's two parts
        seen = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float2 ml = ct.ml[i >> 2][(i & 3) * 32 + lane];
          const float li = ml.y == -1.f ? 0.f : ml.y;
          seen |= ml.y != 0.f;
          // a part whose maximum is -inf holds no weight (or NaN)
          const float f = ml.x == -INFINITY ? (li == 0.f ? 0.f : li)
                                            : ex2(ml.x * a.c - mc);
          lsum += li * f;
          if ((i & 3) == part) {
            if ((i >> 2) == w)
              f1 = f;
            else
              f2 = f;
          }
        }
        if (steps) {
          mbar_wait(smem_u32(&ct.o_full[w]), o_phase, give_up);
          o_phase ^= 1;
        }
        if (steps2) {
          mbar_wait(smem_u32(&ct.o_full[w ^ 1]), o_phase2, give_up);
          o_phase2 ^= 1;
        }
        tc_fence_after();
        // what a CTA that gave up computed is no result
        if (*give_up) lsum = NAN;
        const bool empty = lsum == 0.f;
        const float inv = empty ? 0.f : 1.f / lsum;
        const float fill =
            part == 0 && ((empty && seen && sg.part < 0) || lsum != lsum)
                ? NAN : 0.f;
        f1 *= inv;
        f2 *= inv;
        if (!steps || empty) f1 = 0.f;
        if (!steps2 || empty) f2 = 0.f;
        // A part of no weight is multiplied like the others: 0 * inf shows.
        // Each warpgroup joins half of the columns: [part][row][column],
        // 16-byte pieces permuted by the row so that lanes hit all banks.
        constexpr int kCols = D / 2, kPieces = kCols / 4;
        float4 *join = reinterpret_cast<float4 *>(
                           smem + (1 + Sh::kSlots) * Sh::kTileBytes) +
                       w * 4 * 16 * kPieces;
#pragma unroll 1
        for (int col = 0; col < kCols; col += 32) {
          float o[32];
          uint32_t u[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = fill;
          if (steps) {
            tc_ld32(u, tm_o + w * kCols + col);
            tc_wait_ld();
            tc_hold(u);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = fmaf(__uint_as_float(u[e]), f1, o[e]);
          }
          if (steps2) {
            tc_ld32(u, lane_base + 256 + (w ^ 1) * 128 + w * kCols + col);
            tc_wait_ld();
            tc_hold(u);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              o[e] = fmaf(__uint_as_float(u[e]), f2, o[e]);
          }
          if (row_on) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              join[(part * 16 + lane) * kPieces +
                   ((col / 4 + e) ^ (lane & (kPieces - 1)))] =
                  make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2],
                              o[4 * e + 3]);
          }
        }
        if (row_on && part == 0 && w == 0) {
          const float lse =
              empty ? seen && sg.part >= 0 ? kNoWeight : -INFINITY
                    : mm * a.scale + logf(lsum * kUnshift);
          if (sg.part >= 0)
            a.part_lse[(int64_t)sg.part * kTile + lane] = lse;
          else
            a.lse[(int64_t)(sg.tok0 + tok) * a.l_tok +
                  (int64_t)head * a.l_head] = lse;
        }
        tc_fence_before();
        asm volatile("bar.sync %0, 128;" ::"r"(2 + w) : "memory");
        for (int i = threadIdx.x & 127; i < sg.rows * kPieces; i += 128) {
          const int row = i / kPieces, piece = i % kPieces;
          float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float4 v = join[(q * 16 + row) * kPieces +
                                  (piece ^ (row & (kPieces - 1)))];
            o[0] += v.x;
            o[1] += v.y;
            o[2] += v.z;
            o[3] += v.w;
          }
          const int col = w * kCols + piece * 4;
          const int tk = (sg.row0 + row) / a.group;
          const int hd = sg.hk * a.group + (sg.row0 + row) - tk * a.group;
          if (ct.bad_v)
            give_back<kBf16>(
                o, a.kv, sg, max(sg.t0, masked_from), sg.t1,
                a.tree ? sg.cached : sg.cached + tk + 1,
                a.tree ? a.mask + (int64_t)(sg.tok0 + tk) * a.mask_row
                       : nullptr,
                col);
          if (sg.part >= 0)
            *reinterpret_cast<float4 *>(
                a.part_o + ((int64_t)sg.part * kTile + row) * D + col) =
                make_float4(o[0], o[1], o[2], o[3]);
          else {
            keep_finite<kBf16>(o);
            *reinterpret_cast<uint2 *>(
                a.out + (int64_t)(sg.tok0 + tk) * a.o_tok +
                (int64_t)hd * a.o_head + col * 2) =
                make_uint2(pack16<kBf16>(o[0], o[1]),
                           pack16<kBf16>(o[2], o[3]));
          }
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        continue;
      }
      const bool steps = n_end > t_first;
      bool steps2 = false;                 // the other chain's, if joined
      float m2 = -INFINITY, l2 = 0.f;
      if (kDual) {
        steps2 = w ? true : sg.t1 > sg.t0 + 1;
        ct.ml[w][rt] = make_float2(m, seen && l == 0.f ? -1.f : l);
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float2 other = ct.ml[w ^ 1][rt];
        m2 = other.x;
        l2 = other.y;
        if (l2 == -1.f) {
          seen = true;
          l2 = 0.f;
        }
      }
      if (steps) {
        mbar_wait(smem_u32(&ct.o_full[w]), o_phase, give_up);
        o_phase ^= 1;
      }
      if (kDual && steps2) {
        mbar_wait(smem_u32(&ct.o_full[w ^ 1]), o_phase2, give_up);
        o_phase2 ^= 1;
      }
      tc_fence_after();
      if (warp_on) {
        float mm = kDual ? fmaxf(m, m2) : m;
        const float mc = mm == -INFINITY ? 0.f : mm * a.c;
        // a half whose maximum is -inf holds no weight (or NaN, which stays)
        float f1 = 1.f, f2 = 0.f, lsum = l;
        if (kDual) {
          f1 = m == -INFINITY ? (l == 0.f ? 0.f : l) : ex2(m * a.c - mc);
          f2 = m2 == -INFINITY ? (l2 == 0.f ? 0.f : l2) : ex2(m2 * a.c - mc);
          lsum = l * f1 + l2 * f2;
        }
        // what a CTA that gave up computed is no result
        if (*give_up) lsum = NAN;
        const bool empty = lsum == 0.f;
        float inv = empty ? 0.f : 1.f / lsum;
        const float fill =
            (empty && seen && sg.part < 0) || lsum != lsum ? NAN : 0.f;
        const float lse =
            empty ? seen && sg.part >= 0 ? kNoWeight : -INFINITY
                  : mm * a.scale + logf(lsum * kUnshift);
        f1 *= inv;
        f2 *= inv;
        if (!steps || empty) f1 = 0.f;
        if (!kDual || !steps2 || empty) f2 = 0.f;
        const bool fix = ct.bad_v != 0;
        // two-tile form: each warpgroup writes half of the columns
        constexpr int kCols = kDual ? D / 2 : D;
        const int c_base = kDual ? w * kCols : 0;
        const int64_t prow =
            (int64_t)sg.part * (Sh::kQTiles * kTile) + r;
        char *orow = a.out + (int64_t)(sg.tok0 + tok) * a.o_tok +
                     (int64_t)head * a.o_head;
#pragma unroll 1
        for (int col = c_base; col < c_base + kCols; col += 16) {
          float o[16];
          uint32_t u[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = fill;
          if (steps) {
            tc_ld16(u, tm_o + col);
            tc_wait_ld();
            tc_hold(u);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = fmaf(__uint_as_float(u[e]), f1, o[e]);
          }
          if (kDual && steps2) {
            tc_ld16(u, lane_base + 256 + (w ^ 1) * 128 + col);
            tc_wait_ld();
            tc_hold(u);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              o[e] = fmaf(__uint_as_float(u[e]), f2, o[e]);
          }
          if (row_on) {
            if (fix)
              give_back<kBf16>(o, a.kv, sg, max(sg.t0, masked_from),
                               kDual ? sg.t1 : n_end, lim, mrow, col);
            uint32_t v[8];
            if (sg.part >= 0) {
              float *dst = a.part_o + prow * D + col;
#pragma unroll
              for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  v[e] = __float_as_uint(o[8 * i + e]);
                store32(dst + 8 * i, v, true);
              }
            } else {
              keep_finite<kBf16>(o);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                v[e] = pack16<kBf16>(o[2 * e], o[2 * e + 1]);
              store32(orow + col * 2, v, a.out32);
            }
          }
        }
        if (row_on && (!kDual || w == 0)) {
          if (sg.part >= 0)
            a.part_lse[prow] = lse;
          else
            a.lse[(int64_t)(sg.tok0 + tok) * a.l_tok +
                  (int64_t)head * a.l_head] = lse;
        }
      }
      tc_fence_before();
      if (kDual) asm volatile("bar.sync 1, 256;" ::: "memory");
    }
  } else if (warp < 12) {
    // ------------------------------------------------------- loaders
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    constexpr int kChunks = D / 8;                 // 16-byte chunks of a row
    constexpr int kRowsPer = 32 / kChunks;         // rows per warp step
    const int lw = warp - 8;
    const int chunk = lane % kChunks, sub_row = lane / kChunks;
    uint32_t item = 0, q_phase = 1;

    // Chunk `chunk` of row `row` of a tile, in the 128-byte swizzle.
    auto place = [&](int row) {
      return (uint32_t)((chunk >> 3) * (kTile * 128) + row * 128 +
                        (((chunk & 7) ^ (row & 7)) << 4));
    };
    // A V tile in which some row does not see every key: a key that a row
    // does not see must not reach it through 0 * inf, so inf and NaN go in
    // as zeros (and are added back for the rows that see them, in the
    // epilogue).  Each thread looks at what it copied.
    auto check_finite = [&](uint32_t dst) {
      cp_async_wait_all();
      const uint32_t ex = kBf16 ? 0x7f807f80u : 0x7c007c00u;
      for (int i = 0; i < 32 / kRowsPer; ++i) {
        const uint32_t at = dst + place(lw * 32 + i * kRowsPer + sub_row);
        uint32_t v[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                     : "r"(at)
                     : "memory");
        uint32_t bad = 0;
        for (int e = 0; e < 4; ++e) {
          const uint32_t x = v[e] & ex;
          uint32_t keep = 0;
          if ((x & 0xffffu) != (ex & 0xffffu)) keep |= 0xffffu;
          if ((x >> 16) != (ex >> 16)) keep |= 0xffff0000u;
          bad |= ~keep;
          v[e] &= keep;
        }
        if (bad) {
          ct.bad_v = 1;
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at),
                       "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
                       : "memory");
        }
      }
      fence_async_proxy();
    };
    // A tile is full when every thread's copies have landed (128 arrivals
    // by the copies themselves) and every warp's plain writes are released
    // (4): no thread waits for its own copies, so as many tiles are in
    // flight as there are free slots.
    auto publish = [&](uint32_t bar) {
      cp_async_arrive(bar);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    // One tile: lane `i` of the warp holds the address of its row i (0: the
    // row is not there and reads as zeros).
    auto copy_rows = [&](uint32_t dst, const char *row_ptr) {
#pragma unroll 4
      for (int i = 0; i < 32 / kRowsPer; ++i) {
        const int rl = i * kRowsPer + sub_row;
        const uint64_t p =
            __shfl_sync(0xffffffffu, (uint64_t)row_ptr, rl);
        const char *src = p ? (const char *)p + chunk * 16 : a.q;
        cp_async16(dst + place(lw * 32 + rl), src, p ? 16 : 0);
      }
    };

    auto load_q = [&](const Segment &sg) {
      if (!mbar_wait_warp(smem_u32(&ct.q_empty), q_phase, give_up))
        return false;
      q_phase ^= 1;
      for (int qt = 0; qt < Sh::kQTiles; ++qt) {
        const int r = kFew ? lane : qt * kTile + lw * 32 + lane;
        const char *src = nullptr;
        if (r < sg.rows) {
          const int tok = (sg.row0 + r) / a.group;
          const int head =
              sg.hk * a.group + (sg.row0 + r) - tok * a.group;
          src = a.q + (int64_t)(sg.tok0 + tok) * a.q_tok +
                (int64_t)head * a.q_head;
        }
        copy_rows(sm_q + qt * Sh::kTileBytes, src);
      }
      publish(smem_u32(&ct.q_full));
      return true;
    };

    uint32_t tile_no = 0;
    bool on = true;                      // no wait was let through
    for (int si = seg_begin; si < seg_end && on; ++si) {
      const Segment sg = segs[si];
      const int t_all = kDual ? sg.t1 : max(sg.n0, sg.n1);
      const int masked_from = first_masked_tile(sg, a.group, a.tree);
      // K and V tiles
      const int total = sg.cached + sg.n_new;
      auto page_at = [&](int t) {        // the page of this lane's key
        const int key = t * kTile + lw * 32 + lane;
        return key < sg.cached ? table_entry(a.kv, sg.b, key) : -1;
      };
      int entry = page_at(sg.t0);
      for (int t = sg.t0; t < t_all; ++t) {
        // Q goes behind a tile or two of its segment: it has to wait until
        // the segment before is through with its own, they do not.
        if (t == (si == seg_begin ? sg.t0
                                  : min(sg.t0 + Sh::kAhead, t_all - 1)))
          on = load_q(sg);
        const int key = t * kTile + lw * 32 + lane;
        const int page = page_named(a.kv, entry);
        const char *kp = nullptr, *vp = nullptr;
        if (key < sg.cached) {
          if (page >= 0) {
            const int off = key % a.kv.page;
            kp = a.kv.kp + page * a.kv.kp_page + sg.hk * a.kv.kp_head +
                 off * a.kv.kp_tok;
            vp = a.kv.vp + page * a.kv.vp_page + sg.hk * a.kv.vp_head +
                 off * a.kv.vp_tok;
          }
        } else if (key < total) {
          const int64_t n = sg.tok0 + key - sg.cached;
          kp = a.kv.k + n * a.kv.k_tok + sg.hk * a.kv.k_head;
          vp = a.kv.v + n * a.kv.v_tok + sg.hk * a.kv.v_head;
        }
        if (t + 1 < t_all) entry = page_at(t + 1);
        const uint32_t there = __ballot_sync(0xffffffffu, kp != nullptr);
        // Tiles of one kind that every row sees whole go by TMA.
        const bool by_page = maps.pages_ok && (t + 1) * kTile <= sg.cached;
        const bool by_new = maps.new_ok && t * kTile >= sg.cached &&
                            (t + 1) * kTile <= total && t < masked_from;
        const int tok = sg.tok0 + t * kTile - sg.cached + lw * 32;
        const int off = key % a.kv.page;
#pragma unroll 1
        for (int h = 0; h < 2 && on; ++h) {          // K, V
          const uint32_t slot = item % Sh::kSlots;
          const uint32_t ph = (item / Sh::kSlots) & 1;
          const uint32_t bar = smem_u32(&ct.full[slot]);
          const uint32_t dst = sm_ring + slot * Sh::kTileBytes;
          on = mbar_wait_warp(smem_u32(&ct.empty[slot]), ph ^ 1, give_up);
          if (!on) break;
          if (h == 0 && lane == 0) ct.valid[tile_no & 7][lw] = there;
          if (by_page) {
            fetch_pages<D>(dst + lw * 32 * 128, maps, h ? &maps.vp : &maps.kp,
                           page, off, a.kv.pages, sg.hk, bar, 33);
          } else if (by_new) {
            fetch_new<D>(dst + lw * 32 * 128, h ? &maps.v : &maps.k, tok,
                         sg.hk, bar, 33);
          } else {
            copy_rows(dst, h ? vp : kp);
            if (h == 1 && t >= masked_from) check_finite(dst);
            publish(bar);
          }
          ++item;
        }
        if (!on) break;
        ++tile_no;
      }
    }
    cp_async_wait_all();
    end_copies<Sh::kSlots>(ct.full, ct.sent, lw, item, 33);
  } else {
    // ------------------------------------------------------------ MMA
    // Two row tiles: one warp for each of the two chains S -> P -> O.  A
    // tcgen05.mma holds its warp until the tensor pipe takes it, so whatever a
    // warp does between two of them is time in which only the other warp's
    // MMAs run.  The warps take turns, a step's PV and next QK at a time: MMAs
    // that interleave slow each other down several times over, and both
    // chains fall into step, exponentials under exponentials and MMAs under
    // MMAs (16384 tokens: 5.44 ms against 3.98).
    //
    // Two key tiles, where HBM is the bound: one warp issues whatever is
    // ready next of either chain.
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp < (kDual ? 13 : 14)) {
      const int w = uniform(warp - 12);
      // one lane issues, none once a wait was let through
      uint32_t issue = lane == 0;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!mbar_wait_warp(bar, parity, give_up)) issue = 0;
      };
      const uint32_t tm_s = uniform(tmem) + w * 128, tm_o = tm_s + 256;
      const uint32_t q = tile_desc(
          uniform(sm_q) + (kDual ? 0 : w * Sh::kTileBytes), 0);
      const uint32_t ring = uniform(sm_ring);
      constexpr uint32_t id_qk = mma_idesc(kBf16, kTile, false);
      constexpr uint32_t id_pv = mma_idesc(kBf16, D, true);
      uint32_t base = 0, q_phase = 0, p_phase = 0;
      uint32_t p_phases = 0;               // two key tiles: a bit a chain
      auto ready = [&](uint32_t bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
        if (!__any_sync(0xffffffffu, *give_up != 0)) return false;
        issue = 0;
        return true;
      };
      uint32_t turn_phase = w ^ 1;          // warp 0 has the first turn
      const int seg_last = uniform(seg_end);
      for (int si = uniform(seg_begin); si < seg_last; ++si) {
        const Segment *sp = segs + si;
        const int t0 = uniform(sp->t0);
        const int n0 = uniform(kDual ? sp->t1 : sp->n0);
        const int n1 = uniform(kDual ? sp->t1 : sp->n1);
        const int t_all = max(n0, n1), n_end = w ? n1 : n0;
        const int t_first = t0;
        wait(smem_u32(&ct.q_full), q_phase);
        q_phase ^= 1;
        auto full = [&](uint32_t item) {
          return smem_u32(&ct.full[item % Sh::kSlots]);
        };
        auto phase = [&](uint32_t item) { return (item / Sh::kSlots) & 1; };
        if constexpr (kDual) {
          int tq = t0, tp = t0;            // next S and next O product
          uint32_t rounds = 0;
          while (tp < t_all) {
            bool idle = true;
            const uint32_t k_item = base + 2 * (tq - t0);
            const uint32_t v_item = base + 2 * (tp - t0) + 1;
            // S's buffer is free once the product with its last P is issued
            if (tq < t_all && tq < tp + 2 &&
                ready(full(k_item), phase(k_item))) {
              const int h = (tq - t0) & 1;
              const uint32_t slot = k_item % Sh::kSlots;
              fence_async_proxy();
              tc_fence_after();
              mma_rows<0, D / 16>(tm_s + h * 128, q,
                                  tile_desc(ring + slot * Sh::kTileBytes, 0),
                                  id_qk, issue);
              tc_commit(smem_u32(&ct.s_full[h]), issue);
              tc_commit(smem_u32(&ct.empty[slot]), issue);
              // Q is free for the next segment's from here on
              if (++tq == t_all) tc_commit(smem_u32(&ct.q_empty), issue);
              idle = false;
            }
            const int h = (tp - t0) & 1;
            if (tp < tq &&
                ready(smem_u32(&ct.p_full[h]), (p_phases >> h) & 1) &&
                ready(full(v_item), phase(v_item))) {
              const uint32_t slot = v_item % Sh::kSlots;
              fence_async_proxy();
              tc_fence_after();
              mma_keys<0, kTile / 16>(
                  tm_o + h * 128, tm_s + h * 128,
                  tile_desc(ring + slot * Sh::kTileBytes, kTile * 128), id_pv,
                  tp >= t0 + 2, issue);
              tc_commit(smem_u32(&ct.empty[slot]), issue);
              if (tp + 2 >= t_all) tc_commit(smem_u32(&ct.o_full[h]), issue);
              p_phases ^= 1u << h;
              ++tp;
              idle = false;
            }
            if (idle)
              give_up_after(&rounds, give_up);
            else
              rounds = 0;
          }
          base += 2 * (t_all - t0);
          continue;
        }
        auto pass_turn = [&]() {
          if (issue) mbar_arrive(smem_u32(&ct.turn[w ^ 1]));
        };
        if (t_first < n_end) {
          const uint32_t item = base + 2 * (t_first - t0);
          const uint32_t slot = item % Sh::kSlots;
          wait(full(item), phase(item));
          fence_async_proxy();
          mma_rows<0, D / 16>(tm_s, q,
                              tile_desc(ring + slot * Sh::kTileBytes, 0),
                              id_qk, issue);
          tc_commit(smem_u32(&ct.s_full[w]), issue);
          tc_commit(smem_u32(&ct.empty[slot]), issue);
        }
        // Q is free for the next segment's once the last product with it is
        // done, long before this segment is
        if (t_first + 1 >= n_end) tc_commit(smem_u32(&ct.q_empty), issue);
        for (int t = t_first; t < t_all; ++t) {
          if (t >= n_end) {
            // A tile that only the other row tile needs: give it back, pass
            // the turn on.
            for (int h = 0; h < 2; ++h) {
              const uint32_t item = base + 2 * (t - t0) + h;
              wait(full(item), phase(item));
              if (issue)
                mbar_arrive(smem_u32(&ct.empty[item % Sh::kSlots]));
            }
            wait(smem_u32(&ct.turn[w]), turn_phase);
            turn_phase ^= 1;
            pass_turn();
            continue;
          }
          const uint32_t v_item = base + 2 * (t - t0) + 1;
          const uint32_t k_item = v_item + 1;
          const uint32_t slot = v_item % Sh::kSlots;
          const uint32_t k_slot = k_item % Sh::kSlots;
          const bool more = t + 1 < n_end;
          wait(full(v_item), phase(v_item));
          const uint32_t v =
              tile_desc(ring + slot * Sh::kTileBytes, kTile * 128);
          const uint32_t k = tile_desc(ring + k_slot * Sh::kTileBytes, 0);
          const bool k_there =
              more && __all_sync(0xffffffffu,
                                 mbar_try(full(k_item), phase(k_item)));
          fence_async_proxy();
          wait(smem_u32(&ct.p_full[w]), p_phase);
          p_phase ^= 1;
          wait(smem_u32(&ct.turn[w]), turn_phase);
          turn_phase ^= 1;
          tc_fence_after();
          mma_keys<0, kTile / 16>(tm_o, tm_s, v, id_pv, t != t_first, issue);
          if (!k_there) {
            pass_turn();
            if (!more) tc_commit(smem_u32(&ct.o_full[w]), issue);
            tc_commit(smem_u32(&ct.empty[slot]), issue);
            if (!more) continue;
            wait(full(k_item), phase(k_item));
            fence_async_proxy();
          }
          mma_rows<0, D / 16>(tm_s, q, k, id_qk, issue);
          if (k_there) {
            pass_turn();
            tc_commit(smem_u32(&ct.empty[slot]), issue);
          }
          tc_commit(smem_u32(&ct.s_full[w]), issue);
          tc_commit(smem_u32(&ct.empty[k_slot]), issue);
          if (t + 2 == n_end) tc_commit(smem_u32(&ct.q_empty), issue);
        }
        base += 2 * (t_all - t0);
      }
      // TMEM is freed only when no MMA is in flight.
      tc_commit(smem_u32(&ct.done), lane == 0);
      int ran_out = 0;
      mbar_wait_warp(smem_u32(&ct.done), 0, &ran_out);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tc_dealloc(tmem, 512);
  }
}

// Joins the partial results of items that several CTAs worked on: one warp
// per row, weights exp(lse_p - max lse), in the order of the parts.  It reads a
// few megabytes, mostly from L2; launched early, it is there when the parts
// are, so that what it costs is one round trip.  A part's weight is __expf's:
// off by 2 + 1.2 |x| units in the last place (x = lse_p - max lse), so by less
// than 2^-18 of a weight of e^-16 or more, and smaller ones count for less; an
// output is rounded by 2^-11 or 2^-8.
template <int D, bool kBf16>
__global__ void __launch_bounds__(256)
    attn_merge_kernel(const __grid_constant__ FwdArgs a, const Merge *merges,
                      int slot_rows) {
  wait_for_previous();
  const Merge mg = merges[blockIdx.y];
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (r >= mg.rows) return;
  const int64_t row0 = (int64_t)mg.part0 * slot_rows + r;
  float top = -INFINITY;
  for (int p = lane; p < mg.parts; p += 32)
    top = fmaxf(top, a.part_lse[row0 + (int64_t)p * slot_rows]);
#pragma unroll
  for (int o = 16; o; o >>= 1)
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  constexpr int kPer = D / 32;
  float acc[kPer] = {}, total = 0.f;
  for (int p = 0; p < mg.parts; ++p) {
    const int64_t row = row0 + (int64_t)p * slot_rows;
    const float lse = a.part_lse[row];
    // a part without weight is 0, or NaN where it saw values that are not
    // finite, which stays
    const float wgt = lse <= kNoWeight ? 0.f : __expf(lse - top);
    total += wgt;
    const float *src = a.part_o + row * D + lane * kPer;
#pragma unroll
    for (int e = 0; e < kPer; ++e) acc[e] = fmaf(src[e], wgt, acc[e]);
  }
  // no part has any weight (a NaN is one): 0, or NaN where keys were seen
  const bool none = total == 0.f;
  const float inv = none ? 0.f : 1.f / total;
  const float fill = none && top == kNoWeight ? NAN : 0.f;
  const int tok = (mg.row0 + r) / a.group;
  const int head = mg.hk * a.group + (mg.row0 + r) - tok * a.group;
  char *dst = a.out + (int64_t)(mg.tok0 + tok) * a.o_tok +
              (int64_t)head * a.o_head + lane * kPer * 2;
#pragma unroll
  for (int e = 0; e < kPer; ++e) acc[e] = fmaf(acc[e], inv, fill);
  keep_finite<kBf16>(acc);
#pragma unroll
  for (int e = 0; e < kPer; e += 2)
    *reinterpret_cast<uint32_t *>(dst + e * 2) =
        pack16<kBf16>(acc[e], acc[e + 1]);
  if (lane == 0)
    a.lse[(int64_t)(mg.tok0 + tok) * a.l_tok + (int64_t)head * a.l_head] =
        none ? -INFINITY : top + logf(total);
}

template <int D, bool kBf16, int kForm>
int run_fwd(const FwdArgs &a, const TileMaps &maps,
            const cascade_attn_plan_info_t &p, cudaStream_t s) {
  using Sh = Shape<D, kForm>;
  auto *kernel = attn_fwd_kernel<D, kBf16, kForm>;
  // setmaxnreg hands the launch's registers from the loaders and the MMA
  // warps to the softmax warps: 256 x 192 + 128 x 72 + 128 x 56 = 512 x 128.
  // A launch with fewer would wait for ever, so it is refused.
  static std::atomic<uint64_t> done{0};
  OncePerDevice once(&done);
  if (once.pending()) {
    cudaFuncAttributes fa;
    CB_CUDA(cudaFuncGetAttributes(&fa, kernel));
    CB_CHECK(fa.numRegs == 128, CASCADE_ERR_UNSUPPORTED,
             "attention kernel built with an unexpected register count");
    CB_CUDA(cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
    once.set();
  }
  // early: the blocks are there, barriers set, when the kernel before ends
  // (8 prompts up to 1500 tokens: 146.9 us a pass against 148.7; 8 trees of 64
  // drafts 73.3 against 75.6)
  CB_CUDA(launch_early(kernel, dim3(p.ctas), dim3(kThreads), Sh::kSmem, s, a,
                       maps));
  count_launches(1);
  if (p.merges > 0) {
    const Merge *merges = reinterpret_cast<const Merge *>(
        a.plan + seg_offset(p.ctas) + (int64_t)p.segments * 16);
    const dim3 grid((unsigned)div_up(p.merge_rows, 8), (unsigned)p.merges);
    CB_CUDA(launch_early(attn_merge_kernel<D, kBf16>, grid, dim3(256), 0, s,
                         a, merges, Sh::kQTiles * kTile));
    count_launches(1);
  }
  return CASCADE_OK;
}

}  // namespace
}  // namespace attn
}  // namespace cb

extern "C" int cascade_attn_forward(const cascade_attn_plan_info_t *plan,
                                    const cascade_attn_args_t *args,
                                    void *stream) {
  using namespace cb::attn;
  cb::clear_error();
  CB_CHECK(plan && args, CASCADE_ERR_INVALID, "null pointer argument");
  const cascade_attn_plan_info_t &p = *plan;
  CB_CHECK(p.kind == CASCADE_ATTN_FORWARD, CASCADE_ERR_INVALID,
           "the plan is not one for attention");
  CB_CHECK(args->dtype == CASCADE_KV_FP16 || args->dtype == CASCADE_KV_BF16,
           CASCADE_ERR_INVALID, "dtype must be FP16 or BF16");
  int rc = check_args(p, *args, true);
  if (rc != CASCADE_OK || p.segments == 0) return rc;
  CB_CHECK(args->out && args->lse, CASCADE_ERR_INVALID,
           "null pointer argument");
  CB_CHECK((((uintptr_t)args->out | (uint64_t)(args->out_tok * 2) |
             (uint64_t)(args->out_head * 2)) &
            15) == 0,
           CASCADE_ERR_INVALID, "out must have 16-byte aligned rows");
  CB_CHECK(!p.tree || args->mask, CASCADE_ERR_INVALID,
           "a plan for trees needs a mask");
  CB_CHECK(args->workspace_bytes >= p.workspace_bytes &&
               (p.workspace_bytes == 0 || args->workspace),
           CASCADE_ERR_INVALID, "workspace too small");
  FwdArgs a{};
  fill_source(*args, p, &a.kv);
  a.q = static_cast<const char *>(args->q);
  a.q_tok = args->q_tok * 2;
  a.q_head = args->q_head * 2;
  a.out = static_cast<char *>(args->out);
  a.o_tok = args->out_tok * 2;
  a.o_head = args->out_head * 2;
  a.lse = args->lse;
  a.l_tok = args->lse_tok;
  a.l_head = args->lse_head;
  a.mask = args->mask;
  a.mask_row = args->mask_row;
  a.plan = args->plan;
  const int64_t rows = (int64_t)p.parts * p.row_tile;
  a.part_o = static_cast<float *>(args->workspace);
  a.part_lse = a.part_o + rows * p.head_dim;
  a.ctas = p.ctas;
  a.group = p.q_heads / p.kv_heads;
  a.tree = p.tree;
  a.give_up = diag_give_up();
  a.out32 = (((uintptr_t)args->out | (uint64_t)a.o_tok |
              (uint64_t)a.o_head) &
             31) == 0;
  a.scale = args->scale;
  a.c = args->scale * kLog2e;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = args->dtype == CASCADE_KV_BF16;
  TileMaps maps;
  make_maps(*args, p, true, &maps);
  const int form = p.row_tile > kTile ? kTwoRows
                   : (int64_t)p.max_new * a.group > 16 ? kTwoKeys
                                                       : kFewRows;
  auto run = [&](auto d, auto b) {
    constexpr int kD = decltype(d)::value;
    constexpr bool kB = decltype(b)::value;
    return form == kTwoRows   ? run_fwd<kD, kB, kTwoRows>(a, maps, p, s)
           : form == kTwoKeys ? run_fwd<kD, kB, kTwoKeys>(a, maps, p, s)
                              : run_fwd<kD, kB, kFewRows>(a, maps, p, s);
  };
  using std::integral_constant;
  integral_constant<int, 128> d128;
  integral_constant<int, 64> d64;
  std::true_type yes;
  std::false_type no;
  if (p.head_dim == 128) return bf ? run(d128, yes) : run(d128, no);
  return bf ? run(d64, yes) : run(d64, no);
}

extern "C" int cascade_diag_attn_timeouts(uint64_t *count) {
  using namespace cb::attn;
  cb::clear_error();
  CB_CHECK(count, CASCADE_ERR_INVALID, "null pointer argument");
  void *mine = nullptr;
  CB_CUDA(cudaGetSymbolAddress(&mine, g_timeouts));
  const unsigned int *other = weights_timeouts_symbol();
  CB_CHECK(other, CASCADE_ERR_CUDA, "no device symbol");
  unsigned int v[2] = {0, 0};
  CB_CUDA(cudaMemcpy(&v[0], mine, 4, cudaMemcpyDeviceToHost));
  CB_CUDA(cudaMemcpy(&v[1], other, 4, cudaMemcpyDeviceToHost));
  *count = (uint64_t)v[0] + v[1];
  return CASCADE_OK;
}
