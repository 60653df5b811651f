// Eviction from KV caches: which tokens to keep by their accumulated
// attention weight, and the gather that makes the shorter caches.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.cuh"

namespace cb {
namespace {

namespace cg = cooperative_groups;

struct SelectArgs {
  const float *w;
  int64_t stride[3];               // elements, of the three row dimensions
  int dim1, dim2;                  // rows are (i0 * dim1 + i1) * dim2 + i2
  const int32_t *lengths;          // per i0, or null: all `width`
  int width, budget, recent, sink;
  int32_t *keep;                   // [rows][budget]
};

// Unsigned integers in the order of the weights: -0 equals 0, and NaN ranks
// with -inf, below every number.
__device__ __forceinline__ uint32_t order_of(float w) {
  uint32_t u = __float_as_uint(w);
  if (w != w) u = 0xff800000u;
  if (u == 0x80000000u) u = 0;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One cluster per row of weights; each CTA takes one slice of the row, each
// warp consecutive weights of that, kept in registers (kKeys a lane; 0: a
// row too long for that is read again, from L2, in every round).  The
// need-th largest weight is built from the top, a bit a round: the weights
// that reach the longer prefix are counted, and the counts added up over the
// CTA and, through distributed shared memory, the cluster.  The search ends
// when a prefix has exactly the weights wanted.  Equal weights (a row of
// zeros, the common case after a long prompt) cost what different ones do;
// histograms in shared memory took longer (112 us for 1024 rows of 8192),
// since their atomics pass about one lane a cycle.  Then one ordered pass
// writes the positions above the weight found, and the lowest positions of
// those equal to it.  Bound by instructions: 2 a weight and round, 20 to 32
// rounds; 1024 rows of 8192 take 57 us from HBM, 53 from L2, of which the
// search is half.
template <int kThreads, int kKeys>
__global__ void __launch_bounds__(kThreads, kThreads == 512   ? 3
                                      : kThreads == 1024 ? 1
                                                         : 8)
    evict_select_kernel(const __grid_constant__ SelectArgs a) {
  constexpr int kWarps = kThreads / 32;
  wait_for_previous();
  let_next_start();
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks();
  const int rank = (int)cluster.block_rank();
  __shared__ uint32_t warp_sum[2][kWarps];
  __shared__ uint2 warp_count[2][kWarps];
  __shared__ uint32_t cta_sum[2];
  __shared__ uint32_t cta_total[2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t row = blockIdx.x / (uint32_t)ranks;
  const uint32_t i01 = row / (uint32_t)a.dim2;
  const uint32_t i2 = row - i01 * a.dim2, i0 = i01 / (uint32_t)a.dim1;
  const uint32_t i1 = i01 - i0 * a.dim1;
  const float *w = a.w + i0 * a.stride[0] + i1 * a.stride[1] +
                   i2 * a.stride[2];
  int32_t *keep = a.keep + (int64_t)row * a.budget;
  int len = a.width;
  if (a.lengths != nullptr) len = min(max(a.lengths[i0], 0), a.width);
  const int kept = min(len, a.budget);
  for (int i = kept + rank * kThreads + tid; i < a.budget;
       i += ranks * kThreads)
    keep[i] = -1;
  if (len <= a.budget) {           // the same for the whole cluster
    for (int i = rank * kThreads + tid; i < len; i += ranks * kThreads)
      keep[i] = i;
    return;
  }
  // candidates are [sink, len - recent); the rest is kept anyway
  const int lo = a.sink, hi = len - a.recent;
  const int n = hi - lo;
  const uint32_t need = a.budget - a.sink - a.recent;
  for (int i = rank * kThreads + tid; i < lo; i += ranks * kThreads)
    keep[i] = i;
  for (int i = rank * kThreads + tid; i < a.recent; i += ranks * kThreads)
    keep[a.budget - a.recent + i] = hi + i;
  if (need == 0) return;

  // this warp's candidates: per_warp consecutive ones, lane after lane
  const uint32_t warps = ranks * kWarps;
  const int per_warp = ((n + 31u) / 32 + warps - 1) / warps * 32;
  const int64_t first = ((int64_t)rank * kWarps + warp) * per_warp;
  const int begin = (int)(first < n ? first : n);
  const int end = begin + per_warp < n ? begin + per_warp : n;
  // order_of is above 0, so 0 stands for a candidate that is not there
  auto fetch = [&](int i) -> uint32_t {
    return i < end ? order_of(w[lo + i]) : 0u;
  };
  uint32_t key[kKeys > 0 ? kKeys : 1];
  if (kKeys > 0) {
#pragma unroll
    for (int k = 0; k < kKeys; ++k) key[k] = fetch(begin + k * 32 + lane);
  }

  uint32_t least = 0;              // the need-th largest, so far
#pragma unroll 1
  for (int bit = 31, round = 0; bit >= 0; --bit, round ^= 1) {
    const uint32_t t = least | (1u << bit);
    uint32_t c = 0;
    if (kKeys > 0) {
#pragma unroll
      for (int k = 0; k < kKeys; ++k) c += key[k] >= t;
    } else {
      for (int i = begin + lane; i < end; i += 32) c += fetch(i) >= t;
    }
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) warp_sum[round][warp] = c;
    __syncthreads();
    c = __reduce_add_sync(0xffffffffu,
                          lane < kWarps ? warp_sum[round][lane] : 0u);
    if (ranks > 1) {
      if (tid == 0) cta_sum[round] = c;
      cluster.sync();
      c = __reduce_add_sync(
          0xffffffffu,
          lane < ranks ? *cluster.map_shared_rank(&cta_sum[round], lane)
                       : 0u);
    }
    if (c >= need) least = t;
    if (c == need) {               // these and no others: all above t - 1
      least = t - 1;
      break;
    }
  }
  // now: everything above `least`, and the first ones equal to it
  uint32_t above = 0, equal = 0;
  auto tally = [&](uint32_t u) {
    above += __popc(__ballot_sync(0xffffffffu, u > least));
    equal += __popc(__ballot_sync(0xffffffffu, u == least));
  };
  if (kKeys > 0) {
#pragma unroll
    for (int k = 0; k < kKeys; ++k) tally(key[k]);
  } else {
    for (int i = begin; i < end; i += 32) tally(fetch(i + lane));
  }
  __syncthreads();                 // the counts of the last round are read
  if (lane == 0) warp_count[0][warp] = make_uint2(above, equal);
  __syncthreads();
  if (warp == 0) {
    uint2 v = lane < kWarps ? warp_count[0][lane] : make_uint2(0u, 0u);
    uint32_t x = v.x, y = v.y;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t px = __shfl_up_sync(0xffffffffu, x, o);
      const uint32_t py = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += px;
        y += py;
      }
    }
    if (lane < kWarps) warp_count[1][lane] = make_uint2(x - v.x, y - v.y);
    if (lane == 31) {
      cta_total[0] = x;
      cta_total[1] = y;
    }
  }
  if (ranks > 1)
    cluster.sync();
  else
    __syncthreads();
  uint32_t x = warp_count[1][warp].x, y = warp_count[1][warp].y;
  uint32_t all_above = cta_total[0];
  if (ranks > 1) {
    uint32_t vx = 0, vy = 0, va = 0;
    if (lane < ranks) {
      const uint32_t *o = cluster.map_shared_rank(cta_total, lane);
      va = o[0];
      if (lane < rank) {
        vx = va;
        vy = o[1];
      }
    }
    x += __reduce_add_sync(0xffffffffu, vx);
    y += __reduce_add_sync(0xffffffffu, vy);
    all_above = __reduce_add_sync(0xffffffffu, va);
  }
  const uint32_t equals = need - all_above;   // how many of the equal ones
  auto write = [&](uint32_t u, int i) {
    const uint32_t below = (1u << lane) - 1;
    const uint32_t gt = __ballot_sync(0xffffffffu, u > least);
    const uint32_t eq = __ballot_sync(0xffffffffu, u == least);
    const uint32_t my_eq = y + __popc(eq & below);
    const uint32_t at = x + __popc(gt & below) + min(my_eq, equals);
    if (u > least || (u == least && my_eq < equals))
      keep[a.sink + at] = lo + i;
    x += __popc(gt);
    y += __popc(eq);
  };
  if (kKeys > 0) {
#pragma unroll
    for (int k = 0; k < kKeys; ++k) write(key[k], begin + k * 32 + lane);
  } else {
    for (int i = begin; i < end; i += 32) write(fetch(i + lane), i + lane);
  }
  if (ranks > 1) cluster.sync();   // the others read this CTA's totals
}

// ------------------------------------------------------------------ gather
constexpr int kGThreads = 256;
constexpr int kGRows = 4;          // rows in flight per thread

// The descriptors travel as kernel parameters, so a call needs no copy to
// the device: 1024 of them (24 KiB) at most, or 16 in the small form, whose
// launch is cheaper.
template <int kTensors>
struct GatherArgs {
  const int32_t *keep;             // [items / layers][heads][kept]
  char *out;                       // [items][2][heads][kept][row bytes]
  const int32_t *table;            // paged sources: [items][table_row]
  int64_t table_row, stride_page;  // the latter in bytes
  int32_t table_cols, page, pages;
  int32_t seq;                     // tokens of an unpaged source
  int32_t heads, kept, per_row;    // vectors of a row
  int32_t item0, layers;
  cascade_kv_tensor_t t[kTensors]; // strides in bytes
};

// One thread copies one vector of each of kGRows kept rows; a block takes
// rows of one head of one tensor.  Bound by HBM: a row of head_dim values is
// contiguous, so its bytes move as full sectors wherever it lies (1.07 GB of
// 256-byte rows in 186 us, 5.8 TB/s; 2 rows in flight took 1.27 times as long,
// 8 1.46 times).
template <typename V, int kTensors>
__global__ void __launch_bounds__(kGThreads)
    evict_gather_kernel(const __grid_constant__ GatherArgs<kTensors> a) {
  const int head = blockIdx.y % a.heads, ti = blockIdx.y / a.heads;
  const int item = a.item0 + (ti >> 1);
  const cascade_kv_tensor_t t = a.t[ti];
  const int32_t *keep =
      a.keep + ((int64_t)(item / a.layers) * a.heads + head) * a.kept;
  const char *base = reinterpret_cast<const char *>(t.ptr) +
                     (int64_t)head * t.stride_head;
  V *out = reinterpret_cast<V *>(a.out) +
           (((int64_t)2 * a.item0 + ti) * a.heads + head) * a.kept *
               (int64_t)a.per_row;
  // threads of a row, rows of a step (a long row takes several steps)
  const int width = min(a.per_row, kGThreads);
  const int step = kGThreads / width;
  const int row_in = threadIdx.x / width, c0 = threadIdx.x - row_in * width;
  const int64_t r0 = (int64_t)blockIdx.x * step * kGRows + row_in;
  if (row_in >= step) return;
  wait_for_previous();             // which may be what chose the rows
  const char *src[kGRows];
#pragma unroll
  for (int i = 0; i < kGRows; ++i) {
    const int64_t r = r0 + i * step;
    src[i] = nullptr;
    if (r >= a.kept) continue;
    const int pos = keep[r];
    if (a.table != nullptr) {
      if (pos >= 0 && pos / a.page < a.table_cols) {
        const int id =
            a.table[(int64_t)item * a.table_row + pos / a.page];
        if (id >= 0 && id < a.pages)
          src[i] = base + id * a.stride_page +
                   (int64_t)(pos % a.page) * t.stride_seq;
      }
    } else if (pos >= 0 && pos < a.seq) {
      src[i] = base + (int64_t)pos * t.stride_seq;
    }
  }
  for (int c = c0; c < a.per_row; c += width) {
    V v[kGRows];
#pragma unroll
    for (int i = 0; i < kGRows; ++i)
      v[i] = src[i] ? reinterpret_cast<const V *>(src[i])[c] : V{};
#pragma unroll
    for (int i = 0; i < kGRows; ++i) {
      const int64_t r = r0 + i * step;
      if (r < a.kept) out[r * a.per_row + c] = v[i];
    }
  }
}

template <int kTensors>
int run_gather(GatherArgs<kTensors> &a, const cascade_kv_tensor_t *src,
               uint32_t tensors, uint32_t elem, int vec, uint32_t step_max,
               unsigned blocks, cudaStream_t s) {
  if (step_max > (uint32_t)kTensors) step_max = kTensors;
  for (uint32_t t0 = 0; t0 < tensors; t0 += step_max) {
    const uint32_t n = tensors - t0 < step_max ? tensors - t0 : step_max;
    a.item0 = (int)(t0 / 2);
    for (uint32_t i = 0; i < n; ++i) {
      a.t[i] = src[t0 + i];
      a.t[i].stride_head *= elem;
      a.t[i].stride_seq *= elem;
    }
    const dim3 grid(blocks, n * a.heads), block(kGThreads);
    if (vec == 16)
      CB_CUDA(launch_early(evict_gather_kernel<uint4, kTensors>, grid, block,
                           0, s, a));
    else if (vec == 4)
      CB_CUDA(launch_early(evict_gather_kernel<uint32_t, kTensors>, grid,
                           block, 0, s, a));
    else
      CB_CUDA(launch_early(evict_gather_kernel<uint16_t, kTensors>, grid,
                           block, 0, s, a));
    count_launches(1);
  }
  return CASCADE_OK;
}

}  // namespace
}  // namespace cb

extern "C" int cascade_kv_evict_select(
    const float *d_weights, const int64_t dims[3], const int64_t strides[3],
    int32_t width, const int32_t *d_lengths, int32_t budget, int32_t recent,
    int32_t sink, int32_t *d_keep, void *stream) {
  using namespace cb;
  clear_error();
  CB_CHECK(dims && strides, CASCADE_ERR_INVALID, "null pointer argument");
  CB_CHECK(dims[0] >= 0 && dims[1] >= 0 && dims[2] >= 0 && width >= 0,
           CASCADE_ERR_INVALID, "negative size");
  CB_CHECK(budget > 0 && recent >= 0 && sink >= 0 &&
               (int64_t)recent + sink <= budget,
           CASCADE_ERR_INVALID,
           "budget must be above 0 and at least recent + sink");
  // positions are stepped along in 32 bits
  CB_CHECK(width <= 1 << 30 && budget <= 1 << 30, CASCADE_ERR_INVALID,
           "rows have at most 2^30 tokens");
  const int64_t big = (int64_t)1 << 27;
  CB_CHECK(dims[0] <= big && dims[1] <= big && dims[2] <= big &&
               dims[0] * dims[1] <= big && dims[0] * dims[1] * dims[2] <= big,
           CASCADE_ERR_INVALID, "too many rows of weights");
  const int64_t rows = dims[0] * dims[1] * dims[2];
  if (rows == 0) return CASCADE_OK;
  CB_CHECK((d_weights || width == 0) && d_keep, CASCADE_ERR_INVALID,
           "null pointer argument");
  SelectArgs a{};
  a.w = d_weights;
  for (int i = 0; i < 3; ++i) a.stride[i] = strides[i];
  a.dim1 = (int)dims[1];
  a.dim2 = (int)dims[2];
  a.lengths = d_lengths;
  a.width = width;
  a.budget = budget;
  a.recent = recent;
  a.sink = sink;
  a.keep = d_keep;
  // A lane holds 4 or 16 weights of a short row (300 weights: 12.3 us for the
  // whole eviction, 18.4 with 512 lanes of 16).  Rows beyond 8192 are spread
  // over clusters of CTAs while there are SMs for them, else over CTAs of
  // 1024 lanes of 32; beyond 8 of those they stay in L2.
  int64_t ranks = 1;
  int threads = 128;
  auto *kernel = evict_select_kernel<128, 4>;
  if (width > 512) kernel = evict_select_kernel<128, 16>;
  if (width > 2048) {
    kernel = evict_select_kernel<512, 16>;
    threads = 512;
  }
  while (ranks * 8192 < width) ranks *= 2;
  if (ranks > 8 || (ranks > 1 && rows * ranks > 2 * sm_count())) {
    threads = 1024;
    ranks = 1;
    while (ranks * 32768 < width) ranks *= 2;
    kernel = ranks <= 8 ? evict_select_kernel<1024, 32>
                        : evict_select_kernel<1024, 0>;
    if (ranks > 8) ranks = 8;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(rows * ranks));
  cfg.blockDim = dim3(threads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ranks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  CB_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
  count_launches(1);
  return CASCADE_OK;
}

extern "C" int cascade_kv_evict_gather(
    const cascade_kv_tensor_t *src, uint32_t items, uint32_t layers,
    uint32_t heads, uint32_t seq, uint32_t head_dim, uint32_t elem_bytes,
    const int32_t *d_keep, uint32_t kept, const int32_t *d_table,
    int64_t table_row, int64_t table_cols, int64_t stride_page, uint32_t page, uint32_t pages,
    void *d_out, void *stream) {
  using namespace cb;
  clear_error();
  CB_CHECK(elem_bytes == 2 || elem_bytes == 4, CASCADE_ERR_INVALID,
           "elements have 2 or 4 bytes");
  CB_CHECK(heads <= 65535 && (uint64_t)head_dim * elem_bytes < (1u << 30) &&
               seq <= INT32_MAX && kept <= INT32_MAX && page <= INT32_MAX &&
               pages <= INT32_MAX && items <= INT32_MAX / 2,
           CASCADE_ERR_INVALID, "a size is out of range");
  CB_CHECK(layers >= 1, CASCADE_ERR_INVALID, "layers must be above 0");
  if (items == 0 || heads == 0 || head_dim == 0 || kept == 0)
    return CASCADE_OK;
  CB_CHECK(src && d_keep && d_out, CASCADE_ERR_INVALID,
           "null pointer argument");
  CB_CHECK(!d_table || (page > 0 && table_cols >= 0), CASCADE_ERR_INVALID,
           "a page table needs a page size");
  // 16-byte vectors when every row starts on a 16-byte boundary, else
  // elements one by one.
  const uint64_t row_bytes = (uint64_t)head_dim * elem_bytes;
  uint64_t bits = (uintptr_t)d_out | row_bytes |
                  (uint64_t)(d_table ? stride_page * elem_bytes : 0);
  const uint32_t tensors = items * 2;
  for (uint32_t i = 0; i < tensors; ++i) {
    CB_CHECK(src[i].ptr || (d_table ? pages == 0 : seq == 0),
             CASCADE_ERR_INVALID, "null pointer argument");
    bits |= src[i].ptr | (uint64_t)(src[i].stride_head * elem_bytes) |
            (uint64_t)(src[i].stride_seq * elem_bytes);
  }
  const int vec = bits & 15 ? (int)elem_bytes : 16;
  const uint32_t per_row = (uint32_t)(row_bytes / vec);
  const uint32_t rows =
      kGThreads / (per_row < kGThreads ? per_row : kGThreads) * kGRows;
  const unsigned blocks = (unsigned)div_up(kept, rows);
  const uint32_t step_max = (65535 / heads) & ~1u;
  CB_CHECK(step_max >= 2, CASCADE_ERR_INVALID, "too many heads");
  auto fill = [&](auto &a) {
    a.keep = d_keep;
    a.out = static_cast<char *>(d_out);
    a.table = d_table;
    a.table_row = table_row;
    a.table_cols = (int)(table_cols < INT32_MAX ? table_cols : INT32_MAX);
    a.stride_page = stride_page * elem_bytes;
    a.page = (int)(page ? page : 1);
    a.pages = (int)pages;
    a.seq = (int)seq;
    a.heads = (int)heads;
    a.kept = (int)kept;
    a.per_row = (int)per_row;
    a.layers = (int)layers;
  };
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (tensors <= 16) {
    GatherArgs<16> a;
    fill(a);
    return run_gather(a, src, tensors, elem_bytes, vec, step_max, blocks, s);
  }
  static thread_local GatherArgs<1024> a;
  fill(a);
  return run_gather(a, src, tensors, elem_bytes, vec, step_max, blocks, s);
}
