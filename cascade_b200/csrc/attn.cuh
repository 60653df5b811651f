// Device pieces shared by the attention kernels (sm_100a): mbarriers with
// bounded waits, tcgen05 / TMEM access, cp.async, and the records that the
// host-side plan hands to the kernels.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace cb {
namespace attn {

// ------------------------------------------------------------------ plan
// The plan buffer is int32: [0, ctas] the first segment of each CTA (and the
// end), padded to 16 ints, then the segments, then the merges.
struct Segment {      // one CTA's consecutive work on one item
  int tok0;           // the sequence's first packed token
  int n_new;          // its new tokens
  int cached;         // its cached tokens
  int b;              // its row of the page table
  int hk;             // key/value head
  int row0;           // first row of the item (row = token * group + head)
  int t0, t1;         // attention: key tiles; weights: row chunks
  int part;           // partial slot, or -1 when the item is whole
  int n0, n1;         // attention: end of the key tiles of either row tile;
                      // weights: n0 pairs of key tiles
  int rows;           // attention: rows of the item
  int key0;           // weights: first key
  int fill;           // weights: the segment ends its sequence's keys
  int pad[2];
};
static_assert(sizeof(Segment) == 64, "segments are 16 ints");

struct Merge {        // one item that several CTAs worked on
  int tok0, hk, row0;
  int rows;           // attention: rows of the item; weights: keys there are
  int part0, parts;
  int b, key0;
};
static_assert(sizeof(Merge) == 32, "merges are 8 ints");

constexpr int kTile = 128;       // keys of a key tile, rows of a row tile

inline __host__ __device__ int seg_offset(int ctas) {
  return (ctas + 1 + 15) / 16 * 16;
}

// --------------------------------------------------------- PTX wrappers
__device__ __forceinline__ uint32_t smem_u32(const void *p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar),
               "r"(count)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar)
               : "memory");
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// The same without being put to sleep for a while: for polling several.
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Waits of this source file's kernels that gave up, on this device.
static __device__ unsigned int g_timeouts;

// A wait on another role of the same CTA.  Every role's loops are finite and
// no address depends on data that a wait guards, so a wait that runs out
// (four million tries, each of which sleeps up to 1.3 us; 5.6 s in all) sets
// the CTA's flag and lets every later wait of the CTA through that is not over
// by itself.  False where it let through: from its own first such wait on a
// warp issues, sends, commits and arrives at nothing more, so that what still
// passes between warps has truly been waited for.  (An arrival that a barrier
// does not expect faults: 2 where 1 is pending.)  The kernel ends by itself,
// its copies waited for (end_copies).  Kept short: it is inlined at every wait.
__device__ __forceinline__ bool mbar_wait_slow(uint32_t bar, uint32_t parity,
                                               volatile int *give_up) {
#pragma unroll 1
  for (uint32_t n = 1; n < (1u << 22); ++n) {
    if (mbar_try(bar, parity)) return true;
    if (*give_up) return false;
  }
  if (*give_up == 0) atomicAdd(&g_timeouts, 1u);
  *give_up = 1;
  return false;
}

__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity,
                                          volatile int *give_up) {
  return mbar_try(bar, parity) || mbar_wait_slow(bar, parity, give_up);
}

// For a loop that polls: gives up when it has had nothing to do for 2^25 rounds
// (over a second; `rounds` starts at 0 and is set back to 0 by progress).
// Counted, as the waits are, and not timed: a process that does not get the
// GPU for a while has waited for nothing.
__device__ __forceinline__ void give_up_after(uint32_t *rounds,
                                              volatile int *give_up) {
  if (++*rounds > (1u << 25) && *give_up == 0) {
    *give_up = 1;
    if ((threadIdx.x & 31) == 0) atomicAdd(&g_timeouts, 1u);
  }
  __syncwarp();
}

// The same for a whole warp, which stays converged.
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity,
                                               volatile int *give_up) {
  if (__all_sync(0xffffffffu, mbar_try(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait_slow(bar, parity, give_up));
}

// The end of the four loader warps, whatever happened: no copy may land in a
// CTA that is gone.  Item i goes to slot i % slots and each warp makes
// `arrivals` of the slot's barrier's for it; a warp that gave up has made
// fewer items than the others.  It makes its arrivals for the rest without
// copies, so that the last phase of every slot completes once all copies have
// landed, and waits for that.  (At most one item a slot is missing: for a
// second, the others would have had to see the first consumed.)
template <int kSlots>
__device__ __forceinline__ void end_copies(const uint64_t *full,
                                           volatile uint32_t *sent, int lw,
                                           uint32_t item, uint32_t arrivals) {
  if ((threadIdx.x & 31) == 0) sent[lw] = item;
  asm volatile("bar.sync 4, 128;" ::: "memory");
  const uint32_t top =
      max(max(sent[0], sent[1]), max(sent[2], sent[3]));
#pragma unroll 1
  for (uint32_t i = item; i < top; ++i)
    if ((threadIdx.x & 31) == 0)
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(
                       smem_u32(&full[i % kSlots])),
                   "r"(arrivals)
                   : "memory");
  int ran_out = 0;
#pragma unroll 1
  for (uint32_t i = top > kSlots ? top - kSlots : 0; i < top; ++i)
    mbar_wait_warp(smem_u32(&full[i % kSlots]), (i / kSlots) & 1, &ran_out);
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src,
                                           uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(
                   dst),
               "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.wait_all;" ::: "memory");
}
// Arrives on `bar` (one of its expected arrivals) once every cp.async that
// this thread has issued so far has landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}
// Between generic-proxy writes to shared memory (cp.async among them) that
// this thread made or has seen complete on an mbarrier, and tcgen05.mma
// reading them.
__device__ __forceinline__ void fence_async_proxy() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_alloc(uint32_t smem_dst, uint32_t cols) {
  asm volatile(
      "tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
          smem_dst),
      "r"(cols)
      : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::
                   : "memory");
}
__device__ __forceinline__ void tc_dealloc(uint32_t tmem, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(
                   tmem),
               "r"(cols)
               : "memory");
}
// The MMA warp runs converged, with every value of its loops the same in all
// lanes, and one lane issues: descriptors and addresses then stay in uniform
// registers.  (Issued from a branch that one lane takes, each tcgen05.mma
// first moves its operands there, which took longer than the MMA itself.)
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
  return __reduce_max_sync(0xffffffffu, x);
}

// Arrives on `bar` once every tcgen05.mma the issuing lane issued is done.
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster"
      ".b64 [%0];\n\t}" ::"r"(bar),
      "r"(issue)
      : "memory");
}

// Shared-memory matrix descriptor of a tile in the 128-byte swizzle: rows of
// 64 16-bit values (128 bytes), 8-row groups 1024 bytes apart, further
// 64-value column blocks `lbo` bytes apart (used when the rows run along K).
// The lower word is made here; the upper one (the group stride, the
// descriptor version and the swizzle) is the same for all tiles.
__device__ __forceinline__ uint32_t tile_desc(uint32_t addr, uint32_t lbo) {
  return ((addr & 0x3FFFF) >> 4) | ((lbo >> 4) << 16);
}
#define CB_DESC_HIGH "0x40004040"

// D[128 x N] (+)= A[128 x 16] B[16 x N], A and B in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b,
                                       uint32_t idesc, uint32_t accumulate,
                                       uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 da, {%1, " CB_DESC_HIGH "};\n\t"
      "mov.b64 db, {%2, " CB_DESC_HIGH "};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(
          d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(issue)
      : "memory");
}
// The same with A in TMEM (two 16-bit values a column, one row a lane).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b,
                                       uint32_t idesc, uint32_t accumulate,
                                       uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 db;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 db, {%2, " CB_DESC_HIGH "};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, "
      "p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(issue)
      : "memory");
}

// S[128 x N] = A B^T over D columns: 16-column steps [kStep, kEnd) in turn.
template <int kStep, int kEnd>
__device__ __forceinline__ void mma_rows(uint32_t d, uint32_t a, uint32_t b,
                                         uint32_t idesc, uint32_t issue) {
#pragma unroll
  for (int k = kStep; k < kEnd; ++k) {
    const uint32_t off = ((k >> 2) * (kTile * 128) + (k & 3) * 32) >> 4;
    mma_ss(d, a + off, b + off, idesc, k, issue);
  }
}
// O[128 x N] (+)= P[128 x 128] V over the key steps [kStep, kEnd).
template <int kStep, int kEnd>
__device__ __forceinline__ void mma_keys(uint32_t d, uint32_t p, uint32_t v,
                                         uint32_t idesc, bool accumulate,
                                         uint32_t issue) {
#pragma unroll
  for (int k = kStep; k < kEnd; ++k)
    mma_ts(d, p + k * 8, v + k * (2048 >> 4), idesc,
           accumulate || k != kStep, issue);
}

// kind::f16 instruction descriptor: 128 x n, FP32 accumulator; `mn_b` when
// B's rows run along K (its columns are contiguous).
__host__ __device__ constexpr uint32_t mma_idesc(bool bf16, int n,
                                                 bool mn_b) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
         ((mn_b ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTile >> 4) << 24);
}

#define CB_R8(x, i)                                                          \
  "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]),                \
      "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define CB_I8(x, i)                                                          \
  "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]),     \
      "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
#define CB_K8(x, i)                                                          \
  "+r"(x[i]), "+r"(x[i + 1]), "+r"(x[i + 2]), "+r"(x[i + 3]),                \
      "+r"(x[i + 4]), "+r"(x[i + 5]), "+r"(x[i + 6]), "+r"(x[i + 7])

// 32 consecutive columns of this warp's 32 lanes; complete after tc_wait_ld.
__device__ __forceinline__ void tc_ld32(uint32_t (&x)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31}, [%32];"
      : CB_R8(x, 0), CB_R8(x, 8), CB_R8(x, 16), CB_R8(x, 24)
      : "r"(addr));
}
__device__ __forceinline__ void tc_st32(uint32_t addr,
                                        const uint32_t (&x)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, "
      "%30, %31};" ::CB_I8(x, 0),
      CB_I8(x, 8), CB_I8(x, 16), CB_I8(x, 24), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t addr,
                                        const uint32_t (&x)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15};" ::CB_I8(x, 0),
      CB_I8(x, 8), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_ld8(uint32_t (&x)[8], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : CB_R8(x, 0)
      : "r"(addr));
}
__device__ __forceinline__ void tc_ld16(uint32_t (&x)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : CB_R8(x, 0), CB_R8(x, 8)
      : "r"(addr));
}
__device__ __forceinline__ void tc_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// Keeps uses of the loaded values behind the wait that completes them.
__device__ __forceinline__ void tc_hold(uint32_t (&x)[32]) {
  asm volatile("" : CB_K8(x, 0), CB_K8(x, 8), CB_K8(x, 16), CB_K8(x, 24));
}

__device__ __forceinline__ void tc_hold(uint32_t (&x)[8]) {
  asm volatile("" : CB_K8(x, 0));
}
__device__ __forceinline__ void tc_hold(uint32_t (&x)[16]) {
  asm volatile("" : CB_K8(x, 0), CB_K8(x, 8));
}

// 32 bytes of one thread: one full sector, where the address allows it.
__device__ __forceinline__ void store32(void *dst, const uint32_t (&v)[8],
                                        bool aligned) {
  if (aligned) {
    asm volatile(
        "st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
        "r"(v[6]), "r"(v[7])
        : "memory");
  } else {
    uint4 *d = static_cast<uint4 *>(dst);
    d[0] = make_uint4(v[0], v[1], v[2], v[3]);
    d[1] = make_uint4(v[4], v[5], v[6], v[7]);
  }
}

// 2^x by the special-function unit: within 2 units in the last place (2^-22 of
// the value), and results below 2^-126 are 0.  The rounding of a score of 16 to
// FP32 alone moves its weight by as much.  One instruction a score: the
// exponentials bound these kernels, and a polynomial of degree 5 on the FMA
// pipe took as many cycles.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two floats to two 16-bit values in one word, to nearest even.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if (kBf16)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// FP16 outputs: a mean of values lies within the type's range, but P's
// rounding can take it 2^-11 beyond the largest value, which would round to
// infinity.  Infinities themselves stay.
template <bool kBf16, int kN>
__device__ __forceinline__ void keep_finite(float (&o)[kN]) {
  if (kBf16) return;
  float top = 0.f;
#pragma unroll
  for (int e = 0; e < kN; ++e) top = fmaxf(top, fabsf(o[e]));
  if (top <= 65504.f) return;
#pragma unroll
  for (int e = 0; e < kN; ++e)
    if (fabsf(o[e]) < INFINITY) o[e] = fminf(fmaxf(o[e], -65504.f), 65504.f);
}

// Pairs of floats in one register pair: one instruction works on both (and
// takes half the room in the instruction cache, which is what it is for).
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float &lo, float &hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// 2^(x c + d) of a pair, joined to `sum`; returns the two rounded to 16 bits.
template <bool kBf16>
__device__ __forceinline__ uint32_t weigh2(uint32_t x0, uint32_t x1,
                                           uint64_t c, uint64_t d,
                                           uint64_t &sum) {
  float y0, y1;
  unpair(fma2(pair_of(__uint_as_float(x0), __uint_as_float(x1)), c, d), y0,
         y1);
  y0 = ex2(y0);
  y1 = ex2(y1);
  sum = add2(sum, pair_of(y0, y1));
  return pack16<kBf16>(y0, y1);
}

constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------- where a key's row is
struct KvSource {
  const char *k, *v;               // new tokens, packed
  int64_t k_tok, k_head, v_tok, v_head;               // strides in bytes
  const char *kp, *vp;             // pages
  int64_t kp_page, kp_head, kp_tok, vp_page, vp_head, vp_tok;
  const int32_t *table;
  int64_t table_row;               // entries between rows of the table
  int32_t page, pages;             // tokens of a page, pages there are
};

// Checks of a call's pointers, alignment and strides (host).
int check_args(const cascade_attn_plan_info_t &p,
               const cascade_attn_args_t &a, bool forward);
void fill_source(const cascade_attn_args_t &a,
                 const cascade_attn_plan_info_t &p, KvSource *s);

unsigned int *weights_timeouts_symbol();

// Set by cascade_diag_attn_give_up: 1 when this thread's calls are to start
// with their CTAs' flag up.
int diag_give_up();

// Tensor maps for tiles that TMA can fetch: 64 columns of up to 32 rows of
// one head, in the 128-byte swizzle.  A warp fetches its 32 rows of a tile
// with a few instructions, where cp.async takes 16 of each lane (a decode step
// of 64 sequences: 214 us against 253; prompts on stored pages: 205 against
// 213).
struct TileMaps {
  CUtensorMap kp, vp;              // [page][head][token of the page][d]
  CUtensorMap k, v;                // [token][head][d]
  int pages_ok, new_ok;            // whether they can be used
  int box;                         // rows of a page that one fetch takes
};

// Fills `m` for the call's tensors (the V maps where `with_v`).  Pages of 8,
// 16, 32 or a multiple of 32 tokens can be fetched so; what has strides that
// a tensor map does not take is left to cp.async.
int make_maps(const cascade_attn_args_t &a, const cascade_attn_plan_info_t &p,
              bool with_v, TileMaps *m);

__device__ __forceinline__ void mbar_arrive_n(uint32_t bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(bar),
               "r"(n)
               : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                   bar),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void tma_rows4(uint32_t dst, const CUtensorMap *map,
                                          int x, int y, int z, int w,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx"
      "::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_rows3(uint32_t dst, const CUtensorMap *map,
                                          int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx"
      "::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// One warp's 32 rows of a tile of cached tokens: this lane's key is on page
// `page` (-1: none, which reads as zeros) at token `off`.  Arrives on `bar`
// like `plain` arrivals of the cp.async form.
template <int D>
__device__ __forceinline__ void fetch_pages(uint32_t dst, const TileMaps &m,
                                            const CUtensorMap *map, int page,
                                            int off, int pages, int hk,
                                            uint32_t bar, uint32_t plain) {
  const int lane = threadIdx.x & 31;
  constexpr int kHalves = D / 64;
  if (lane == 0) {
    mbar_expect(bar, 32 * D * 2);
    mbar_arrive_n(bar, plain - 1);
  }
  __syncwarp();
  const int piece = lane / kHalves, half = lane % kHalves;
  const int row = piece * m.box;
  const int pg = __shfl_sync(0xffffffffu, page, row & 31);
  const int tok = __shfl_sync(0xffffffffu, off, row & 31);
  if (row < 32)
    tma_rows4(dst + half * (kTile * 128) + row * 128, map, half * 64, tok, hk,
              pg < 0 ? pages : pg, bar);
}
// The same for new tokens from packed token `tok` on.
template <int D>
__device__ __forceinline__ void fetch_new(uint32_t dst, const CUtensorMap *map,
                                          int tok, int hk, uint32_t bar,
                                          uint32_t plain) {
  const int lane = threadIdx.x & 31;
  if (lane == 0) {
    mbar_expect(bar, 32 * D * 2);
    mbar_arrive_n(bar, plain - 1);
  }
  __syncwarp();
  if (lane < D / 64)
    tma_rows3(dst + lane * (kTile * 128), map, lane * 64, hk, tok, bar);
}

// The table's entry for cached token `key` of sequence b, and the page that
// it names (-1: none).  Apart, so that an entry can be on its way while other
// work is done: it is waited for where it is first looked at.  A plain load:
// the non-coherent path is for memory that nothing writes during the kernel's
// life, and an early launch may live beside the kernel that writes the table.
__device__ __forceinline__ int table_entry(const KvSource &s, int b,
                                           int key) {
  return s.table[(int64_t)b * s.table_row + key / s.page];
}
__device__ __forceinline__ int page_named(const KvSource &s, int id) {
  return id >= 0 && id < s.pages ? id : -1;
}
__device__ __forceinline__ int page_of(const KvSource &s, int b, int key) {
  return page_named(s, table_entry(s, b, key));
}

}  // namespace attn
}  // namespace cb
