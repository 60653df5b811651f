// The host side of the attention operators: plans (which CTA does which part
// of a batch) and the checks of a call's arguments.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstring>
#include <exception>
#include <queue>
#include <vector>

#include "attn.cuh"

namespace cb {
namespace attn {

int check_args(const cascade_attn_plan_info_t &p,
               const cascade_attn_args_t &a, bool forward) {
  CB_CHECK(p.segments == 0 || a.plan, CASCADE_ERR_INVALID,
           "null pointer argument");
  CB_CHECK(((uintptr_t)a.plan & 15) == 0 &&
               ((uintptr_t)a.workspace & 31) == 0,
           CASCADE_ERR_INVALID,
           "the plan must be 16-byte, the workspace 32-byte aligned");
  // (the kernels work with scale log2(e) and 8 / that)
  CB_CHECK(a.scale >= 0x1p-64f && a.scale <= 0x1p64f, CASCADE_ERR_INVALID,
           "scale must be in [2^-64, 2^64]");
  uint64_t bits = (uintptr_t)a.q | (uintptr_t)a.k;
  int64_t strides = a.q_tok | a.q_head | a.k_tok | a.k_head;
  if (forward) {
    bits |= (uintptr_t)a.v;
    strides |= a.v_tok | a.v_head;
  }
  CB_CHECK(p.tokens == 0 || (a.q && a.k && (a.v || !forward)),
           CASCADE_ERR_INVALID, "null pointer argument");
  if (p.max_cached > 0) {
    // (no pages at all have no address)
    CB_CHECK(a.table && a.pages >= 0 &&
                 (a.pages == 0 || (a.k_pages && (a.v_pages || !forward))),
             CASCADE_ERR_INVALID, "cached tokens need pages and a table");
    bits |= (uintptr_t)a.k_pages;
    strides |= a.kp_page | a.kp_head | a.kp_tok;
    if (forward) {
      bits |= (uintptr_t)a.v_pages;
      strides |= a.vp_page | a.vp_head | a.vp_tok;
    }
  }
  CB_CHECK((bits & 15) == 0 && (strides & 7) == 0, CASCADE_ERR_INVALID,
           "rows of q, k, v and the pages must start on 16-byte boundaries");
  return CASCADE_OK;
}

void fill_source(const cascade_attn_args_t &a,
                 const cascade_attn_plan_info_t &p, KvSource *s) {
  s->k = static_cast<const char *>(a.k);
  s->v = static_cast<const char *>(a.v);
  s->k_tok = a.k_tok * 2;
  s->k_head = a.k_head * 2;
  s->v_tok = a.v_tok * 2;
  s->v_head = a.v_head * 2;
  s->kp = static_cast<const char *>(a.k_pages);
  s->vp = static_cast<const char *>(a.v_pages);
  s->kp_page = a.kp_page * 2;
  s->kp_head = a.kp_head * 2;
  s->kp_tok = a.kp_tok * 2;
  s->vp_page = a.vp_page * 2;
  s->vp_head = a.vp_head * 2;
  s->vp_tok = a.vp_tok * 2;
  s->table = a.table;
  s->table_row = a.table_row;
  s->page = p.page_size > 0 ? p.page_size : 1;
  s->pages = a.pages;
}

namespace {

thread_local int give_up = 0;

}  // namespace

int diag_give_up() { return give_up; }

namespace {

using EncodeTiled = decltype(&cuTensorMapEncodeTiled);

EncodeTiled encode_tiled() {
  static std::atomic<EncodeTiled> cached{nullptr};
  EncodeTiled fn = cached.load(std::memory_order_acquire);
  if (fn == nullptr) {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000,
                                         cudaEnableDefault, &found) ==
            cudaSuccess &&
        found == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiled>(p);
    cached.store(fn, std::memory_order_release);
  }
  return fn;
}

// A map of 64 x rows boxes; sizes and strides (in elements) from the second
// dimension on.  False when the driver does not take them.
bool encode(CUtensorMap *m, const void *base, int head_dim, int rank,
            const int64_t *size, const int64_t *stride, int box_dim, int rows,
            int dtype) {
  cuuint64_t dims[4] = {(cuuint64_t)head_dim}, bytes[3];
  cuuint32_t box[4] = {64, 1, 1, 1}, step[4] = {1, 1, 1, 1};
  for (int i = 0; i + 1 < rank; ++i) {
    // a dimension of one element is never stepped along
    const int64_t s = size[i] == 1 ? head_dim : stride[i];
    if (size[i] <= 0 || size[i] > (1ll << 31) || s <= 0 ||
        s >= (1ll << 38))
      return false;
    dims[i + 1] = (cuuint64_t)size[i];
    bytes[i] = (cuuint64_t)s * 2;
  }
  box[box_dim] = (cuuint32_t)rows;
  const EncodeTiled fn = encode_tiled();
  return fn != nullptr &&
         fn(m,
            dtype == CASCADE_KV_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
            (cuuint32_t)rank, const_cast<void *>(base), dims, bytes, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

int make_maps(const cascade_attn_args_t &a, const cascade_attn_plan_info_t &p,
              bool with_v, TileMaps *m) {
  std::memset(m, 0, sizeof(*m));
  const int page = p.page_size;
  if (p.max_cached >= kTile && a.pages > 0 &&
      (page == 8 || page == 16 || (page > 0 && page % 32 == 0))) {
    m->box = page < 32 ? page : 32;
    const int64_t size[3] = {page, p.kv_heads, a.pages};
    const int64_t ks[3] = {a.kp_tok, a.kp_head, a.kp_page};
    const int64_t vs[3] = {a.vp_tok, a.vp_head, a.vp_page};
    m->pages_ok =
        encode(&m->kp, a.k_pages, p.head_dim, 4, size, ks, 1, m->box,
               a.dtype) &&
        (!with_v || encode(&m->vp, a.v_pages, p.head_dim, 4, size, vs, 1,
                           m->box, a.dtype));
  }
  if (p.max_new >= kTile) {
    const int64_t size[2] = {p.kv_heads, p.tokens};
    const int64_t ks[2] = {a.k_head, a.k_tok}, vs[2] = {a.v_head, a.v_tok};
    m->new_ok =
        encode(&m->k, a.k, p.head_dim, 3, size, ks, 2, 32, a.dtype) &&
        (!with_v ||
         encode(&m->v, a.v, p.head_dim, 3, size, vs, 2, 32, a.dtype));
  }
  return CASCADE_OK;
}

namespace {

struct Item {
  Segment seg;       // t0, t1: its whole range of units
  int units() const { return seg.t1 - seg.t0; }
};

// Time per unit (a key tile, or a chunk of rows) and per segment, and what a
// merge costs, in nanoseconds.  They decide between splits only; results do
// not depend on them beyond the order in which partial sums are joined.
struct Costs {
  double unit, unit_bytes, segment, merge, part_bytes;
};

constexpr double kBytesPerNs = 6200;       // HBM, all SMs together
constexpr double kPartBytesPerNs = 35;     // partial results, one SM

Merge merge_of(const Segment &s, bool fwd, int part0, int parts) {
  Merge m{};
  m.tok0 = s.tok0;
  m.hk = s.hk;
  m.row0 = s.row0;
  m.rows = fwd ? s.rows : s.n_new + s.cached;
  m.part0 = part0;
  m.parts = parts;
  m.b = s.b;
  m.key0 = s.key0;
  return m;
}

// Items longer than `cap` units are cut into equal pieces; the pieces go, the
// longest first, each to the CTA with the least to do.
std::vector<std::vector<Segment>> cut_items(const std::vector<Item> &items,
                                            int ctas, int cap, bool fwd,
                                            const Costs &c,
                                            std::vector<Merge> *merges,
                                            int *parts, double *makespan) {
  std::vector<Segment> pieces;
  pieces.reserve(items.size());
  for (const Item &it : items) {
    const int n = std::max(1, (int)div_up(it.units(), cap));
    if (n > 1) merges->push_back(merge_of(it.seg, fwd, *parts, n));
    for (int k = 0; k < n; ++k) {
      Segment s = it.seg;
      s.t0 = it.seg.t0 + (int)((int64_t)it.units() * k / n);
      s.t1 = it.seg.t0 + (int)((int64_t)it.units() * (k + 1) / n);
      if (n > 1) s.part = (*parts)++;
      pieces.push_back(s);
    }
  }
  std::vector<int> order(pieces.size());
  for (size_t i = 0; i < order.size(); ++i) order[i] = (int)i;
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) {
    return pieces[x].t1 - pieces[x].t0 > pieces[y].t1 - pieces[y].t0;
  });
  ctas = (int)std::min<size_t>(ctas, pieces.size());
  std::vector<std::vector<Segment>> out(ctas);
  using Load = std::pair<double, int>;
  std::priority_queue<Load, std::vector<Load>, std::greater<Load>> heap;
  for (int i = 0; i < ctas; ++i) heap.push({0.0, i});
  const double unit = std::max(c.unit, c.unit_bytes * ctas / kBytesPerNs);
  double longest = 0;
  for (int i : order) {
    Load l = heap.top();
    heap.pop();
    const Segment &s = pieces[i];
    l.first += (s.t1 - s.t0) * unit + c.segment +
               (s.part >= 0 ? c.part_bytes / 2 / kPartBytesPerNs : 0);
    longest = std::max(longest, l.first);
    out[l.second].push_back(s);
    heap.push(l);
  }
  *makespan = longest + (*parts ? c.merge + *parts * c.part_bytes / 2 /
                                                4000.0
                                : 0);
  return out;
}

// Cuts the items, laid end to end, into `ctas` equal runs.
std::vector<std::vector<Segment>> equal_runs(const std::vector<Item> &items,
                                             int ctas, const Costs &c,
                                             bool fwd,
                                             std::vector<Merge> *merges,
                                             int *parts) {
  const double ov = c.segment / c.unit;
  double total = 0;
  for (const Item &it : items) total += it.units() + ov;
  const double quota = total / ctas;
  std::vector<std::vector<Segment>> out(ctas);
  double pos = 0;
  int cta = 0;
  std::vector<std::pair<int, size_t>> pieces;       // (CTA, its segment)
  for (const Item &it : items) {
    const int units = it.units();
    int done = 0;
    pieces.clear();
    do {
      // units of this item in front of the end of this CTA's run
      const double room = (cta + 1) * quota - pos - ov / 2;
      int end = units;
      if (cta < ctas - 1)
        end = (int)std::lround(
            std::min(std::max(room, (double)done), (double)units));
      if (end > done || units == 0) {
        Segment s = it.seg;
        s.t0 = it.seg.t0 + done;
        s.t1 = it.seg.t0 + end;
        pieces.push_back({cta, out[cta].size()});
        out[cta].push_back(s);
        done = end;
      }
      if (done < units) ++cta;
    } while (done < units);
    if (pieces.size() > 1) {
      merges->push_back(merge_of(it.seg, fwd, *parts, (int)pieces.size()));
      for (const auto &at : pieces) out[at.first][at.second].part = (*parts)++;
    }
    pos += units + ov;
    while (cta < ctas - 1 && pos >= (cta + 1) * quota) ++cta;
  }
  return out;
}

int make_plan(cascade_attn_plan_info_t *info, const int32_t *n_new,
              const int32_t *n_cached, int32_t *buf, size_t capacity) {
  cascade_attn_plan_info_t &p = *info;
  const bool fwd = p.kind == CASCADE_ATTN_FORWARD;
  const int group = p.q_heads / p.kv_heads;
  const int sms = p.sms > 0 ? p.sms : sm_count();
  int64_t tokens = 0;
  int max_new = 0, max_cached = 0, max_keys = 0;
  for (int b = 0; b < p.batch; ++b) {
    const int c = n_cached ? n_cached[b] : 0;
    CB_CHECK(n_new[b] >= 0 && c >= 0, CASCADE_ERR_INVALID,
             "lengths must not be negative");
    CB_CHECK((int64_t)n_new[b] + c <= (1 << 30), CASCADE_ERR_INVALID,
             "a sequence has at most 2^30 tokens");
    CB_CHECK((int64_t)n_new[b] * group <= (1 << 30), CASCADE_ERR_INVALID,
             "a sequence has at most 2^30 query rows");
    tokens += n_new[b];
    max_new = std::max(max_new, n_new[b]);
    max_cached = std::max(max_cached, c);
    max_keys = std::max(max_keys, n_new[b] + c);
  }
  CB_CHECK(tokens <= (1 << 30), CASCADE_ERR_INVALID,
           "at most 2^30 packed tokens");
  CB_CHECK(max_cached == 0 || p.page_size > 0, CASCADE_ERR_INVALID,
           "cached tokens need a page size");
  p.tokens = tokens;
  p.max_new = max_new;
  p.max_cached = max_cached;
  p.max_keys = max_keys;
  p.table_cols =
      p.page_size > 0 ? (int)div_up(max_cached, p.page_size) : 0;
  // Up to 128 rows fit one row tile: the form for decode.
  const int row_tile =
      !fwd || (int64_t)max_new * group > kTile ? 2 * kTile : kTile;
  p.row_tile = row_tile;

  // Weights of at most 128 rows a sequence: keys stream by the rows.
  const bool by_keys =
      !fwd && (int64_t)std::min(max_new, p.window) * group <= kTile;

  std::vector<Item> items;
  int64_t count = 0, tok0 = 0;
  for (int b = 0; b < p.batch; ++b) {
    const int64_t keys = (int64_t)n_new[b] + (n_cached ? n_cached[b] : 0);
    count += (int64_t)p.kv_heads *
             (fwd ? (int64_t)div_up((uint64_t)n_new[b] * group, row_tile)
                  : std::max<int64_t>(1, (int64_t)div_up(keys, row_tile)));
  }
  CB_CHECK(count <= (1 << 22), CASCADE_ERR_INVALID,
           "the batch is too large for one call");
  items.reserve(count);
  for (int b = 0; b < p.batch; ++b) {
    const int n = n_new[b], c = n_cached ? n_cached[b] : 0;
    for (int hk = 0; hk < p.kv_heads; ++hk) {
      Item it{};
      it.seg.tok0 = (int)tok0;
      it.seg.n_new = n;
      it.seg.cached = c;
      it.seg.b = b;
      it.seg.hk = hk;
      it.seg.part = -1;
      if (fwd) {
        const int rows = n * group;
        // key tiles that the rows up to `last` (not included) see
        auto tiles = [&](int last) {
          const int keys = c + (p.tree ? n : (last - 1) / group + 1);
          return (int)div_up(keys, kTile);
        };
        for (int r = 0; r < rows; r += row_tile) {
          it.seg.row0 = r;
          it.seg.rows = std::min(row_tile, rows - r);
          it.seg.t0 = 0;
          it.seg.n0 = tiles(std::min(rows, r + kTile));
          it.seg.n1 =
              it.seg.rows > kTile ? tiles(std::min(rows, r + row_tile)) : 0;
          it.seg.t1 = std::max(it.seg.n0, it.seg.n1);
          items.push_back(it);
        }
      } else {
        const int w = std::min(n, p.window);
        it.seg.row0 = n - w;              // first token that counts
        it.seg.rows = w * group;
        const int chunks = (int)div_up((uint64_t)it.seg.rows, kTile);
        const int keys = c + n;
        if (by_keys) {
          // one chunk of rows at most: a unit is a pair of key tiles
          it.seg.t0 = 0;
          it.seg.t1 = std::max(1, (int)div_up(keys, row_tile));
          it.seg.n1 = chunks;
          items.push_back(it);
          continue;
        }
        int key = 0;
        it.seg.n0 = 1;
        do {
          // rows of tokens before key - cached see none of these keys
          const int64_t first =
              std::max<int64_t>(0, (int64_t)key - c - it.seg.row0);
          it.seg.key0 = key;
          it.seg.t0 = std::min<int64_t>(chunks, first * group / kTile);
          it.seg.t1 = chunks;
          it.seg.fill = key + row_tile >= keys;
          items.push_back(it);
          key += row_tile;
        } while (key < keys);
      }
    }
    tok0 += n;
  }

  // Time of a unit measured on a B200 (D = 128): a key tile against 256 rows
  // is bound by the exponentials and the MMAs; against one row tile by the
  // latency of one step, or by HBM once all SMs read.
  Costs cost{};
  const double tile_bytes = 2.0 * kTile * p.head_dim;
  if (fwd) {
    cost.unit = row_tile == kTile ? 700 : 2200;
    cost.unit_bytes = row_tile == kTile ? 2 * tile_bytes : 0;
    cost.segment = row_tile == kTile ? 2500 : 5000;
    cost.part_bytes = 8.0 * (p.head_dim + 1) *
                      std::min<int64_t>(row_tile, (int64_t)max_new * group);
  } else {
    const int64_t rows = (int64_t)std::min(max_new, p.window) * group;
    cost.unit = by_keys ? 400 + 800.0 * rows / kTile : 1200;
    cost.unit_bytes = by_keys ? 2 * tile_bytes : 0;
    cost.segment = by_keys ? 500 : 1500;
    cost.part_bytes = by_keys ? 0 : 8.0 * row_tile;
  }
  // a second launch, of which the host's share is the larger; runs of keys
  // need no merge
  cost.merge = by_keys ? 0 : 6000;

  std::vector<std::vector<Segment>> best;
  std::vector<Merge> merges;
  int parts = 0;
  if (!items.empty()) {
    int64_t units = 0;
    int most = 0;
    for (const Item &it : items) {
      units += it.units();
      most = std::max(most, it.units());
    }
    // Whole items, or items cut to a length between the longest's and an
    // equal share's.
    double t_best = 0;
    const int share = (int)std::max<int64_t>(1, units / sms);
    int caps[6] = {std::max(most, 1)}, n_caps = 1;
    if (!by_keys)
      for (int k = 1; k <= 4; ++k) {
        const int cap = std::max(1, share * (k + 3) / 4);
        if (cap < most) caps[n_caps++] = cap;
      }
    for (int k = 0; k < n_caps; ++k) {
      std::vector<Merge> m;
      int n_parts = 0;
      double t;
      auto plan = cut_items(items, sms, caps[k], fwd, cost, &m, &n_parts, &t);
      if (k == 0 || t < t_best * 0.97) {
        t_best = t;
        best.swap(plan);
        merges.swap(m);
        parts = n_parts;
      }
      if (items.size() > 20000) break;      // many items balance by themselves
    }
    // Runs of equal length over n CTAs: where the items are many and HBM is
    // the bound, each CTA then cuts two items at most.
    int n_best = 0;
    if (most > 1) {
      for (int n = sms; n >= 2; n = n * 3 / 4) {
        if (units < n) continue;
        const double unit =
            std::max(cost.unit, cost.unit_bytes * n / kBytesPerNs);
        const double t = (units * unit + items.size() * cost.segment) / n +
                         cost.segment + cost.merge +
                         cost.part_bytes / kPartBytesPerNs +
                         n * cost.part_bytes / 4000.0;
        if (t < t_best * 0.97) {
          t_best = t;
          n_best = n;
        }
      }
    }
    if (n_best) {
      merges.clear();
      parts = 0;
      best = equal_runs(items, n_best, cost, fwd, &merges, &parts);
    }
    if (by_keys) {
      merges.clear();
      parts = 0;
    }
  }
  size_t segments = 0;
  for (const auto &v : best) segments += v.size();
  const size_t ints = (size_t)seg_offset((int)best.size()) + segments * 16 +
                      merges.size() * 8;
  CB_CHECK(ints <= (size_t)INT32_MAX, CASCADE_ERR_INVALID,
           "the batch is too large for one call");
  p.ints = (int)ints;
  p.ctas = (int)best.size();
  p.segments = (int)segments;
  p.parts = parts;
  p.merges = (int)merges.size();
  p.merge_rows = 0;
  for (const Merge &m : merges)
    p.merge_rows = std::max(p.merge_rows, fwd ? m.rows : row_tile);
  p.workspace_bytes =
      (uint64_t)parts * row_tile * (fwd ? p.head_dim + 1 : 1) * 4;
  if (ints > capacity || !buf) return CASCADE_OK;
  std::memset(buf, 0, ints * 4);
  Segment *out = reinterpret_cast<Segment *>(buf + seg_offset(p.ctas));
  int at = 0;
  for (int c = 0; c < p.ctas; ++c) {
    buf[c] = at;
    for (Segment s : best[c]) {
      if (fwd) {
        s.n0 = std::max(s.t0, std::min(s.n0, s.t1));
        s.n1 = std::max(s.t0, std::min(s.n1, s.t1));
      } else if (by_keys) {
        // from units to keys, pairs and the one chunk
        s.key0 = s.t0 * row_tile;
        s.n0 = s.t1 - s.t0;
        s.fill = s.t1 * row_tile >= s.n_new + s.cached;
        s.t0 = 0;
        s.t1 = s.n1;
        s.part = -1;
      }
      out[at++] = s;
    }
  }
  buf[p.ctas] = at;
  if (!merges.empty())
    std::memcpy(out + at, merges.data(), merges.size() * sizeof(Merge));
  return CASCADE_OK;
}

}  // namespace
}  // namespace attn
}  // namespace cb

extern "C" int cascade_attn_plan(cascade_attn_plan_info_t *info,
                                 const int32_t *new_lengths,
                                 const int32_t *cached_lengths, int32_t *out,
                                 size_t capacity) {
  cb::clear_error();
  CB_CHECK(info, CASCADE_ERR_INVALID, "null pointer argument");
  const cascade_attn_plan_info_t &p = *info;
  CB_CHECK(p.kind == CASCADE_ATTN_FORWARD || p.kind == CASCADE_ATTN_WEIGHTS,
           CASCADE_ERR_INVALID, "unknown kind of plan");
  CB_CHECK(p.batch >= 0 && (p.batch == 0 || new_lengths),
           CASCADE_ERR_INVALID, "bad batch");
  CB_CHECK(p.head_dim == 64 || p.head_dim == 128, CASCADE_ERR_INVALID,
           "head_dim must be 64 or 128");
  CB_CHECK(p.kv_heads > 0 && p.q_heads > 0 && p.q_heads % p.kv_heads == 0 &&
               p.q_heads <= 65536,
           CASCADE_ERR_INVALID,
           "q_heads must be a multiple of kv_heads");
  CB_CHECK(p.page_size >= 0 && p.sms >= 0, CASCADE_ERR_INVALID,
           "bad page size or SM count");
  CB_CHECK(p.kind == CASCADE_ATTN_FORWARD || p.window > 0,
           CASCADE_ERR_INVALID, "window must be above 0");
  try {
    return cb::attn::make_plan(info, new_lengths, cached_lengths, out,
                               capacity);
  } catch (const std::exception &) {     // an allocation's, there are no others
    cb::set_error("out of host memory for the plan");
    return CASCADE_ERR_NOMEM;
  }
}

extern "C" void cascade_diag_attn_give_up(int32_t on) {
  cb::attn::give_up = on != 0;
}

extern "C" void cascade_attn_struct_sizes(size_t *plan_info, size_t *args) {
  if (plan_info) *plan_info = sizeof(cascade_attn_plan_info_t);
  if (args) *args = sizeof(cascade_attn_args_t);
}
