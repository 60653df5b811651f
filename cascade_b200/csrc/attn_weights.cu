// Attention weight of every key: the sum over query rows of exp(s - lse).
#include "attn.cuh"
#include "kernels.cuh"

namespace cb {
namespace attn {
namespace {

constexpr int kWThreads = 672;     // 4 x 4 summing warps, 4 loaders, MMA
constexpr int kKeys = 2 * kTile;   // keys of an item
constexpr int kKSlots = 4, kQSlots = 3;   // tiles of 128 keys, of 128 rows

struct WeightArgs {
  KvSource kv;
  const char *q;
  int64_t q_tok, q_head;           // bytes
  const float *lse;
  int64_t l_tok, l_head;
  const float *before;
  int64_t b_seq, b_head;
  float *out;
  int64_t o_seq, o_head;
  const int32_t *plan;
  float *part;                     // [slot][256]
  int ctas, group, width, fill, give_up;
  float c;                         // scale * log2(e)
};

// 2^(x c + d) of a pair, 0 where it is not on.
__device__ __forceinline__ uint64_t exp2_where(uint32_t x0, uint32_t x1,
                                               uint64_t c, uint64_t d,
                                               bool on0, bool on1) {
  float y0, y1;
  unpair(fma2(pair_of(__uint_as_float(x0), __uint_as_float(x1)), c, d), y0,
         y1);
  return pair_of(on0 ? ex2(y0) : 0.f, on1 ? ex2(y1) : 0.f);
}

struct WControl {
  // minus the lse of a chunk's rows, in powers of two
  alignas(16) float lse2[kQSlots][kTile];
  float other[kKeys];              // sums of the odd chunks
  uint64_t k_full[kKSlots], k_empty[kKSlots];
  uint64_t q_full[kQSlots], q_empty[kQSlots];
  uint64_t s_full[2][2], s_empty[2][2];
  uint64_t done;
  uint32_t tmem, sent[4];          // the latter: key tiles of each loader
  int give_up;
};

template <int D>
constexpr int weights_smem() {
  return (kKSlots + kQSlots) * kTile * D * 2 + (int)sizeof(WControl);
}
static_assert(weights_smem<128>() <= 232448, "shared memory of one SM");

// Mathematics.  w_j = sum over the rows r that see key j of
// exp(scale k_j . q_r - lse_r).  The product is formed transposed, S^T =
// K Q^T, with 128 keys as the rows of a tcgen05 tile: a thread owns one key
// and adds along its own row, so the sum over the rows of all heads of a
// group needs no reduction across threads and no atomics, and its order is
// fixed.  A pair of tiles of 128 keys is worked on at a time.  With many query
// rows a segment is one pair that stays resident while chunks of 128 rows stream
// by; with up to 128 rows (a decode step, a short window) it is a run of
// pairs that stream by one resident chunk of N = 32, 64, ... columns.  Key j
// is seen by the rows of tokens from j on, so a thread's mask is one row
// number.  A chunk's sum is taken by itself before it joins the total.
//
// What bounds it (B200, D = 128).  Whole prompts: one exponential per score,
// the special-function unit is 72 % active; 8192 tokens of 32 heads over 8
// take 344 us (369 to 380 in a long run under the power cap), of which the
// exponentials alone are 239.  Decode: HBM; 32 sequences of 4200 tokens read
// 278 MB in 64 us, the launch, the first loads and the last sums included.
template <int D, bool kBf16>
__global__ void __launch_bounds__(kWThreads, 1)
    attn_weights_kernel(const __grid_constant__ WeightArgs a,
                        const __grid_constant__ TileMaps maps) {
  constexpr int kTileBytes = kTile * D * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t sm_k = smem_u32(smem);
  const uint32_t sm_q = sm_k + kKSlots * kTileBytes;
  WControl &ct = *reinterpret_cast<WControl *>(
      smem + (kKSlots + kQSlots) * kTileBytes);
  volatile int *give_up = &ct.give_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (sm_k & 1023) {
    if (threadIdx.x == 0) atomicAdd(&g_timeouts, 1u);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < kKSlots; ++i) {
      mbar_init(smem_u32(&ct.k_full[i]), 128);
      mbar_init(smem_u32(&ct.k_empty[i]), 1);
    }
    for (int i = 0; i < kQSlots; ++i) {
      mbar_init(smem_u32(&ct.q_full[i]), 128 + 4);
      mbar_init(smem_u32(&ct.q_empty[i]), 17);  // the MMAs and 16 warps
    }
    for (int w = 0; w < 2; ++w)
      for (int i = 0; i < 2; ++i) {
        mbar_init(smem_u32(&ct.s_full[w][i]), 1);
        mbar_init(smem_u32(&ct.s_empty[w][i]), 4);
      }
    mbar_init(smem_u32(&ct.done), 1);
    ct.give_up = a.give_up;
    if (a.give_up) atomicAdd(&g_timeouts, 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // The launch may be early: what is in memory may be what the kernel before
  // this one writes, the plan included.  TMEM too is taken behind the wait:
  // a block of that kernel that shares the SM may still have to get its own,
  // and each would wait for the other.  The next kernel may start once it is
  // taken.
  wait_for_previous();
  if (warp == 20) tc_alloc(smem_u32(&ct.tmem), 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  let_next_start();
  const uint32_t tmem = ct.tmem;
  const Segment *segs =
      reinterpret_cast<const Segment *>(a.plan + seg_offset(a.ctas));
  const int seg_begin = a.plan[blockIdx.x], seg_end = a.plan[blockIdx.x + 1];

  if (warp < 16) {
    // ---------------------------------------------------------- sums
    // Two warpgroups for each 128 keys take chunks (or pairs) in turn.
    const int w = (warp >> 2) & 1;
    const uint32_t buf = warp >> 3;
    const int kt = w * kTile + (warp & 3) * 32 + lane;   // key of the item
    const uint32_t tm = tmem + ((uint32_t)((warp & 3) * 32) << 16) + w * 256;
    const uint64_t c2 = pair_of(a.c, a.c);
    uint32_t step = 0, q_no = 0;
    bool on = true;                      // no wait was let through
    for (int si = seg_begin; si < seg_end; ++si) {
      const Segment sg = segs[si];
      const int total = sg.cached + sg.n_new;
      const int64_t hk = sg.hk;
      const float *before =
          a.before != nullptr ? a.before + sg.b * a.b_seq + hk * a.b_head
                              : nullptr;
      float *out = a.out + sg.b * a.o_seq + hk * a.o_head;
      for (int pair = 0; pair < sg.n0; ++pair) {
        // runs of pairs: each is one step, and one warpgroup's of two
        if (sg.n0 > 1 && (sg.t1 > sg.t0 ? step & 1 : 0) != buf) {
          step += sg.t1 - sg.t0;
          continue;
        }
        const int key = sg.key0 + pair * kKeys + kt;
        // on their way while the scores are waited for
        const int entry =
            key < sg.cached ? table_entry(a.kv, sg.b, key) : 0;
        float prev = 0.f;
        if (key < total && before != nullptr) prev = before[key];
        // rows from `from` on see this key
        const int64_t from =
            (int64_t)(key - sg.cached - sg.row0) * a.group;
        float sum = 0.f;
        for (int ch = sg.t0; ch < sg.t1; ++ch, ++step) {
          if ((step & 1) != buf) continue;
          const uint32_t slot = (q_no + ch - sg.t0) % kQSlots;
          const int n = min(kTile, sg.rows - ch * kTile);
          on = mbar_wait(smem_u32(&ct.s_full[w][buf]), (step >> 1) & 1,
                         give_up) &&
               on;
          tc_fence_after();
          const ulonglong2 *l4 =
              reinterpret_cast<const ulonglong2 *>(ct.lse2[slot]);
          const int64_t hidden = from - (int64_t)ch * kTile;
          const bool whole = __all_sync(0xffffffffu, hidden <= 0);
          uint64_t s0 = 0, s1 = 0;
          auto add4 = [&](const uint32_t *x, const ulonglong2 &l) {
            weigh2<false>(x[0], x[1], c2, l.x, s0);
            weigh2<false>(x[2], x[3], c2, l.y, s1);
          };
          const uint32_t src = tm + buf * 128;
          if (whole && n == kTile) {
            // kept short: its code and that of the other warps has to stay
            // in the instruction cache
#pragma unroll 1
            for (int i = 0; i < kTile; i += 32) {
              uint32_t x[32];
              tc_ld32(x, src + i);
              tc_wait_ld();
              tc_hold(x);
#pragma unroll
              for (int e = 0; e < 8; ++e) add4(&x[4 * e], l4[i / 4 + e]);
            }
          } else {
            // few rows, or rows that do not see the key: nothing of those is
            // added, whatever their scores and lse are (NaN included)
#pragma unroll 1
            for (int i = 0; i < n; i += 8) {
              uint32_t x[8];
              tc_ld8(x, src + i);
              tc_wait_ld();
              tc_hold(x);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const ulonglong2 l = l4[i / 4 + e / 2];
                const bool on0 = i + 2 * e >= hidden && i + 2 * e < n;
                const bool on1 = i + 2 * e + 1 >= hidden && i + 2 * e + 1 < n;
                uint64_t &to = e & 1 ? s1 : s0;
                to = add2(to, exp2_where(x[2 * e], x[2 * e + 1], c2,
                                         e & 1 ? l.y : l.x, on0, on1));
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0 && on) {
            mbar_arrive(smem_u32(&ct.s_empty[w][buf]));
            // the chunk is done with after this warpgroup's last pair
            if (sg.n0 == 1)
              mbar_arrive_n(smem_u32(&ct.q_empty[slot]), 2);
            else if (pair + 2 >= sg.n0)
              mbar_arrive(smem_u32(&ct.q_empty[slot]));
          }
          float y0, y1;
          unpair(add2(s0, s1), y0, y1);
          sum += y0 + y1;
        }
        if (sg.n0 == 1) {
          // one pair: its odd and even chunks are joined
          if (buf) ct.other[kt] = sum;
          asm volatile("bar.sync %0, 256;" ::"r"(1 + w) : "memory");
          if (!buf) sum += ct.other[kt];
          asm volatile("bar.sync %0, 256;" ::"r"(1 + w) : "memory");
          if (buf) continue;
        }
        if (key >= total ||
            (key < sg.cached && page_named(a.kv, entry) < 0))
          sum = 0.f;
        if (*give_up) sum = NAN;         // no result
        if (sg.part >= 0)
          a.part[(int64_t)sg.part * kKeys + kt] = sum;
        else if (key < total)
          out[key] = prev + sum;
      }
      q_no += sg.t1 - sg.t0;
      if (sg.fill && a.fill && buf == 0)
        for (int k = total + kt; k < a.width; k += kKeys)
          out[k] = before != nullptr ? before[k] : 0.f;
    }
  } else if (warp < 20) {
    // ------------------------------------------------------- loaders
    constexpr int kChunks = D / 8;
    constexpr int kRowsPer = 32 / kChunks;
    const int lw = warp - 16;
    const int chunk = lane % kChunks, sub_row = lane / kChunks;
    uint32_t k_no = 0, q_no = 0;
    auto place = [&](int row) {
      return (uint32_t)((chunk >> 3) * (kTile * 128) + row * 128 +
                        (((chunk & 7) ^ (row & 7)) << 4));
    };
    auto copy_rows = [&](uint32_t dst, const char *row_ptr) {
#pragma unroll
      for (int i = 0; i < 32 / kRowsPer; ++i) {
        const int rl = i * kRowsPer + sub_row;
        const uint64_t p =
            __shfl_sync(0xffffffffu, (uint64_t)row_ptr, rl);
        const char *src = p ? (const char *)p + chunk * 16 : a.q;
        cp_async16(dst + place(lw * 32 + rl), src, p ? 16 : 0);
      }
    };
    // lse of row r of chunk ch (in powers of two), and its Q row
    auto row_at = [&](const Segment &sg, int ch, const char **src) {
      const int r = lw * 32 + lane, row = ch * kTile + r;
      *src = nullptr;
      if (row >= sg.rows) return -INFINITY;   // a row that counts for nothing
      const int tok = row / a.group;
      const int64_t head = sg.hk * a.group + row - tok * a.group;
      const int64_t at = (int64_t)sg.tok0 + sg.row0 + tok;
      *src = a.q + at * a.q_tok + head * a.q_head;
      const float l = a.lse[at * a.l_tok + head * a.l_head];
      return l == -INFINITY ? -INFINITY : l * -kLog2e;
    };
    auto load_chunk = [&](const Segment &sg, int ch) {
      const uint32_t slot = q_no % kQSlots;
      const char *src;
      const float l2 = row_at(sg, ch, &src);
      if (!mbar_wait_warp(smem_u32(&ct.q_empty[slot]),
                          ((q_no / kQSlots) & 1) ^ 1, give_up))
        return false;
      ct.lse2[slot][lw * 32 + lane] = l2;
      // the MMA reads the rows up to the next multiple of 32
      if (ch * kTile + lw * 32 < sg.rows)
        copy_rows(sm_q + slot * kTileBytes, src);
      // the copies arrive by themselves, the warp for what it wrote
      cp_async_arrive(smem_u32(&ct.q_full[slot]));
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ct.q_full[slot]));
      ++q_no;
      return true;
    };
    bool on = true;                      // no wait was let through
    for (int si = seg_begin; si < seg_end && on; ++si) {
      const Segment sg = segs[si];
      if (sg.t0 >= sg.t1) continue;
      const int total = sg.cached + sg.n_new;
      auto page_at = [&](int tile) {
        const int key = sg.key0 + tile * kTile + lw * 32 + lane;
        return key < sg.cached ? table_entry(a.kv, sg.b, key) : -1;
      };
      const int tiles = 2 * sg.n0;
      // the table is read two tiles ahead
      int entry[2] = {page_at(0), page_at(1)};
      for (int tile = 0; tile < tiles && on; ++tile) {
        const int key = sg.key0 + tile * kTile + lw * 32 + lane;
        const int page = page_named(a.kv, entry[0]);
        const char *kp = nullptr;
        if (key < sg.cached) {
          if (page >= 0)
            kp = a.kv.kp + page * a.kv.kp_page + sg.hk * a.kv.kp_head +
                 (key % a.kv.page) * a.kv.kp_tok;
        } else if (key < total) {
          kp = a.kv.k + (int64_t)(sg.tok0 + key - sg.cached) * a.kv.k_tok +
               sg.hk * a.kv.k_head;
        }
        const int off = key % a.kv.page;
        const int key0 = sg.key0 + tile * kTile;
        const bool by_page = maps.pages_ok && key0 + kTile <= sg.cached;
        const bool by_new =
            maps.new_ok && key0 >= sg.cached && key0 + kTile <= total;
        entry[0] = entry[1];
        if (tile + 2 < tiles) entry[1] = page_at(tile + 2);
        const uint32_t slot = k_no % kKSlots;
        on = mbar_wait_warp(smem_u32(&ct.k_empty[slot]),
                            ((k_no / kKSlots) & 1) ^ 1, give_up);
        if (!on) break;
        const uint32_t bar = smem_u32(&ct.k_full[slot]);
        const uint32_t dst = sm_k + slot * kTileBytes;
        if (by_page) {
          fetch_pages<D>(dst + lw * 32 * 128, maps, &maps.kp, page, off,
                         a.kv.pages, sg.hk, bar, 32);
        } else if (by_new) {
          fetch_new<D>(dst + lw * 32 * 128, &maps.k,
                       sg.tok0 + key0 - sg.cached + lw * 32, sg.hk, bar, 32);
        } else {
          copy_rows(dst, kp);
          cp_async_arrive(bar);
        }
        ++k_no;
        // the first chunk goes behind the first pair: its slot may still
        // have to be freed, theirs are free already
        if (tile == 1) on = load_chunk(sg, sg.t0);
      }
      for (int ch = sg.t0 + 1; ch < sg.t1 && on; ++ch) on = load_chunk(sg, ch);
    }
    cp_async_wait_all();
    end_copies<kKSlots>(ct.k_full, ct.sent, lw, k_no, 32);
  } else {
    // ------------------------------------------------------------ MMA
    {
      // one lane issues, none once a wait was let through
      uint32_t issue = lane == 0;
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!mbar_wait_warp(bar, parity, give_up)) issue = 0;
      };
      const uint32_t tm = uniform(tmem), sk = uniform(sm_k);
      const uint32_t sq = uniform(sm_q);
      uint32_t k_no = 0, step = 0, q_no = 0;
      const int seg_last = uniform(seg_end);
      for (int si = uniform(seg_begin); si < seg_last; ++si) {
        const int t0 = uniform(segs[si].t0), t1 = uniform(segs[si].t1);
        const int rows = uniform(segs[si].rows), pairs = uniform(segs[si].n0);
        if (t0 >= t1) continue;
        for (int pair = 0; pair < pairs; ++pair, k_no += 2) {
          for (int ch = t0; ch < t1; ++ch, ++step) {
            const uint32_t buf = step & 1, qi = q_no + ch - t0;
            const uint32_t slot = qi % kQSlots;
            const int n = min(kTile, (rows - ch * kTile + 31) / 32 * 32);
            const uint32_t idesc = mma_idesc(kBf16, n, false);
            const uint32_t q = tile_desc(sq + slot * kTileBytes, 0);
            if (pair == 0)
              wait(smem_u32(&ct.q_full[slot]), (qi / kQSlots) & 1);
#pragma unroll 1
            for (int w = 0; w < 2; ++w) {
              const uint32_t ks = (k_no + w) % kKSlots;
              if (ch == t0)
                wait(smem_u32(&ct.k_full[ks]), ((k_no + w) / kKSlots) & 1);
              fence_async_proxy();
              wait(smem_u32(&ct.s_empty[w][buf]), ((step >> 1) & 1) ^ 1);
              tc_fence_after();
              mma_rows<0, D / 16>(tm + w * 256 + buf * 128,
                                  tile_desc(sk + ks * kTileBytes, 0), q,
                                  idesc, issue);
              tc_commit(smem_u32(&ct.s_full[w][buf]), issue);
              if (ch + 1 == t1) tc_commit(smem_u32(&ct.k_empty[ks]), issue);
            }
            if (pair + 1 == pairs)
              tc_commit(smem_u32(&ct.q_empty[slot]), issue);
          }
        }
        q_no += t1 - t0;
      }
      tc_commit(smem_u32(&ct.done), lane == 0);
      int ran_out = 0;
      mbar_wait_warp(smem_u32(&ct.done), 0, &ran_out);
    }
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 20) {
    tc_fence_after();
    tc_dealloc(tmem, 512);
  }
}

// Adds the partial sums of items that several CTAs worked on, in order.
__global__ void __launch_bounds__(kKeys)
    weights_merge_kernel(const __grid_constant__ WeightArgs a,
                         const Merge *merges) {
  wait_for_previous();
  const Merge mg = merges[blockIdx.x];
  const int key = mg.key0 + threadIdx.x;
  if (key >= mg.rows) return;
  float sum = 0.f;
  for (int p = 0; p < mg.parts; ++p)
    sum += a.part[(int64_t)(mg.part0 + p) * kKeys + threadIdx.x];
  float prev = 0.f;
  if (a.before != nullptr)
    prev = a.before[mg.b * a.b_seq + (int64_t)mg.hk * a.b_head + key];
  a.out[mg.b * a.o_seq + (int64_t)mg.hk * a.o_head + key] = prev + sum;
}

template <int D, bool kBf16>
int run_weights(const WeightArgs &a, const TileMaps &maps,
                const cascade_attn_plan_info_t &p, cudaStream_t s) {
  auto *kernel = attn_weights_kernel<D, kBf16>;
  constexpr int smem = weights_smem<D>();
  static std::atomic<uint64_t> done{0};
  OncePerDevice once(&done);
  if (once.pending()) {
    CB_CUDA(cudaFuncSetAttribute(
        kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    once.set();
  }
  CB_CUDA(launch_early(kernel, dim3(p.ctas), dim3(kWThreads), smem, s, a,
                       maps));
  count_launches(1);
  if (p.merges > 0) {
    const Segment *segs =
        reinterpret_cast<const Segment *>(a.plan + seg_offset(p.ctas));
    const Merge *merges = reinterpret_cast<const Merge *>(segs + p.segments);
    CB_CUDA(launch_early(weights_merge_kernel, dim3(p.merges), dim3(kKeys), 0,
                         s, a, merges));
    count_launches(1);
  }
  return CASCADE_OK;
}

}  // namespace

unsigned int *weights_timeouts_symbol() {
  void *p = nullptr;
  return cudaGetSymbolAddress(&p, g_timeouts) == cudaSuccess
             ? static_cast<unsigned int *>(p)
             : nullptr;
}

}  // namespace attn
}  // namespace cb

extern "C" int cascade_attn_weights(const cascade_attn_plan_info_t *plan,
                                    const cascade_attn_args_t *args,
                                    void *stream) {
  using namespace cb::attn;
  cb::clear_error();
  CB_CHECK(plan && args, CASCADE_ERR_INVALID, "null pointer argument");
  const cascade_attn_plan_info_t &p = *plan;
  CB_CHECK(p.kind == CASCADE_ATTN_WEIGHTS, CASCADE_ERR_INVALID,
           "the plan is not one for attention weights");
  CB_CHECK(args->dtype == CASCADE_KV_FP16 || args->dtype == CASCADE_KV_BF16,
           CASCADE_ERR_INVALID, "dtype must be FP16 or BF16");
  int rc = check_args(p, *args, false);
  if (rc != CASCADE_OK || p.segments == 0) return rc;
  // no keys, and no positions behind them that are to be written
  if (p.max_keys == 0 && (args->width == 0 || !args->fill)) return rc;
  CB_CHECK(args->weights && (p.tokens == 0 || args->lse),
           CASCADE_ERR_INVALID, "null pointer argument");
  CB_CHECK(args->width >= p.max_keys, CASCADE_ERR_INVALID,
           "rows of weights are shorter than the longest sequence");
  CB_CHECK(!args->add || args->before, CASCADE_ERR_INVALID,
           "null pointer argument");
  CB_CHECK(args->workspace_bytes >= p.workspace_bytes &&
               (p.workspace_bytes == 0 || args->workspace),
           CASCADE_ERR_INVALID, "workspace too small");
  WeightArgs a{};
  fill_source(*args, p, &a.kv);
  a.q = static_cast<const char *>(args->q);
  a.q_tok = args->q_tok * 2;
  a.q_head = args->q_head * 2;
  a.lse = args->lse;
  a.l_tok = args->lse_tok;
  a.l_head = args->lse_head;
  a.before = args->add ? args->before : nullptr;
  a.b_seq = args->before_seq;
  a.b_head = args->before_head;
  a.out = args->weights;
  a.o_seq = args->weights_seq;
  a.o_head = args->weights_head;
  a.plan = args->plan;
  a.part = static_cast<float *>(args->workspace);
  a.ctas = p.ctas;
  a.group = p.q_heads / p.kv_heads;
  a.width = args->width;
  a.fill = args->fill;
  a.give_up = diag_give_up();
  a.c = args->scale * kLog2e;
  TileMaps maps;
  make_maps(*args, p, false, &maps);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf = args->dtype == CASCADE_KV_BF16;
  if (p.head_dim == 128)
    return bf ? run_weights<128, true>(a, maps, p, s)
              : run_weights<128, false>(a, maps, p, s);
  return bf ? run_weights<64, true>(a, maps, p, s) : run_weights<64, false>(a, maps, p, s);
}
