// The step's tables, built on the GPU from the requests' lengths: offsets, key counts, new pages, every row's slot and
// request, the runs of rows that go into one page, and the split of the attention's key tiles over its workers.
//
// Mathematics: four exclusive prefix sums over the requests (rows, new pages, runs, tiles) and, for each row, page, run
// and worker, the request that its index falls into (a binary search in the sums).  Nothing of it depends on the layer,
// so one plan serves a step's every layer.
//
// Bound: latency.  A step of 64 single tokens moves 1.6 KB; what it costs is one launch and a chain of a few dependent
// loads and a block-wide scan.  So one block does it all where the step is small: the sums stay in its shared memory
// and no second launch waits for them.  A large step's rows are written by a second launch over many blocks, which reads
// the sums from the plan.
//
// Measured, on the GPU and as a call (which the host's side bounds below 15 us): 64 single tokens 8.9 and 14.9 us; 128
// windows of 50 tokens 7.0 us, its rows 3.6 more behind it, and 17.4; 256 prompts of up to 4095 tokens (4.3 MB of rows) 11.1,
// its rows 6 more, and 17.2, of which the look at the 16 thousand pages they take is 1.2 (2.7 an entry at a time).  With 1, 4,
// 5 and 25 query heads to a key head such prompts' plans take 17, 17, 24 and 26 us on the GPU: their tile sums' periods.
#include "paged.h"

namespace t2w {

PagedCut paged_cut(int max_fresh, int q_heads, int kv_heads, int head_dim) {
  const int group = q_heads / kv_heads;
  PagedCut c;
  if ((int64_t)max_fresh * group <= 16) {
    c.form = PagedForm::kFew;
    c.part_rows = 16;
    c.tq = max_fresh;
    c.kt = 32;
    c.workers = few_warps * few_blocks(head_dim, max_fresh * group > 8 ? 2 : 1) * num_sms();
    c.min_per = 2;
    c.extra = 4;
    c.whole = false;
  } else if (head_dim == 64 && (int64_t)max_fresh * group <= 16 * mid_warps) {
    // Where one 64-row tile has all of a request's rows and products are short.  Measured (bf16, either form for the same
    // call): 64 requests of 8 tokens, 4 heads to a key head, 40 to 4100 keys: 97 us against 112 to 122 in tiles of 128
    // rows; 128 of 50 tokens, 400 keys: 64 against 66.  With more rows the larger tiles win (32 of 24 tokens, 4 heads, 2000
    // keys: 90 against 56), and with head_dim 128 always (the calls before: 178 against 122, 102 against 77).
    c.form = PagedForm::kMid;
    c.part_rows = 16 * mid_warps;
    c.tq = 16 * mid_warps / group;
    c.kt = 64;
    c.workers = mid_blocks * num_sms();
    c.min_per = 2;
    c.extra = 2;
    c.whole = true;
  } else {
    c.form = PagedForm::kMany;
    c.part_rows = 128;
    c.tq = 128 / group;
    c.kt = 64;
    c.workers = 2 * num_sms();
    c.min_per = 4;
    c.extra = 4;  // (4 chunks of 700 to 1024 tokens over 4096 keys: 136 us with 1, 131 with 2, 130 with 4)
    c.whole = true;
  }
  return c;
}

PlanLayout paged_layout(int64_t requests, int64_t rows, int page, const PagedCut& cut) {
  PlanLayout l;
  l.max_workers = cut.workers;
  int64_t runs = rows / page + 2 * requests;  // a request's rows touch at most two pages more than they fill
  l.max_runs = (int)(runs < rows ? runs : rows);
  int64_t at = sizeof(PlanHead) / 4;
  auto take = [&](int64_t n) {
    const int64_t a = at;
    at += round4(n);
    return a;
  };
  l.q_start = take(requests + 1);
  l.kv_len = take(requests);
  l.slot = take(rows);
  l.request = take(rows);
  l.new_base = take(requests + 1);
  l.run_base = take(requests + 1);
  l.tile_base = take(requests + 1);
  l.seg_base = take(requests + 1);
  l.starts = take(8 * ((int64_t)l.max_workers + 1));
  l.runs = take(4 * (int64_t)l.max_runs);
  l.total = at;
  return l;
}

namespace {

struct PlanDev {
  int requests, rows, max_fresh, page, shift /* page == 1 << shift */, table_ld, max_blocks, pages, causal, kv_heads;
  PagedCut cut;
  PlanLayout lay;
  const int* fresh;
  const int* length;
  int* table;
  const int* free_pages;  // nullptr: the caches do not grow
  const int* free_count;
  int* kv_len_out;        // where the key counts go besides the plan (may be `length`), or nullptr
  int* free_left_out;     // the same for the free count (may be `free_count`)
  int* buf;
  int scattered;          // the rows are written by k_plan_rows
};

struct Sums {
  long long rows, pages, runs, tiles, segs;
};
T2W_DEV Sums add(const Sums& a, const Sums& b) {
  return Sums{a.rows + b.rows, a.pages + b.pages, a.runs + b.runs, a.tiles + b.tiles, a.segs + b.segs};
}
T2W_DEV Sums shfl_up(const Sums& s, int d) {
  return Sums{__shfl_up_sync(~0u, s.rows, d), __shfl_up_sync(~0u, s.pages, d), __shfl_up_sync(~0u, s.runs, d),
              __shfl_up_sync(~0u, s.tiles, d), __shfl_up_sync(~0u, s.segs, d)};
}

// Pages of n tokens.
T2W_DEV int pages_of(int n, int shift) { return (int)(((long long)n + (1 << shift) - 1) >> shift); }

// What request r adds to each sum; false where its lengths are not to be used.
T2W_DEV bool of_request(const PlanDev& p, int f, int len, Sums& s) {
  s = Sums{0, 0, 0, 0, 0};
  if (f < 0 || len < 0 || f > p.max_fresh || (p.free_pages && (long long)len + f > 0x7fffffffLL)) return false;
  const int kv = p.free_pages ? len + f : len;
  if (pages_of(kv, p.shift) > p.max_blocks) return false;
  s.rows = f;
  if (p.free_pages && f > 0) {
    s.pages = pages_of(kv, p.shift) - pages_of(len, p.shift);
    s.runs = pages_of(kv, p.shift) - (len >> p.shift);
  }
  if (f > 0) {
    const int nq = (f + p.cut.tq - 1) / p.cut.tq;
    s.tiles = p.kv_heads * tiles_before(f, kv, p.causal, p.cut.tq, p.cut.kt, nq);
    s.segs = (long long)p.kv_heads * nq;
  }
  return true;
}

// The last i in [0, n) with base[i] <= x (base ascending, base[0] = 0 <= x): zero-wide entries are passed over.
T2W_DEV int find(const int* base, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (base[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// The rows' slots and requests, the new pages' table entries and the runs, items i0, i0 + step, ... of each.
T2W_DEV void scatter(const PlanDev& p, const int* q_start, const int* new_base, const int* run_base, const int* kv_len,
                     int n_rows, int n_pages, int n_runs, int free_n, int i0, int step) {
  int* const slot = p.buf + p.lay.slot;
  int* const request = p.buf + p.lay.request;
  // page of block b of request r: from the free list where it is new in this step (its table entry may not be written yet);
  // k_plan has looked at both
  auto page_of = [&](int r, int b, int len) {
    const int first = pages_of(len, p.shift);
    return b < first ? p.table[(size_t)r * p.table_ld + b] : p.free_pages[free_n - 1 - (new_base[r] + b - first)];
  };
  // four rows in a row at a time: they are mostly of one request and one page
  for (int i = 4 * i0; i < p.rows; i += 4 * step) {
    int r = i < n_rows ? find(q_start, p.requests, i) : -1, page_at = -1, g = 0;
    int s[4], o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[j] = o[j] = -1;
      if (i + j >= n_rows) continue;
      while (i + j >= q_start[r + 1]) {
        ++r;
        page_at = -1;
      }
      o[j] = r;
      if (!p.free_pages) continue;
      const int len = kv_len[r] - (q_start[r + 1] - q_start[r]), pos = len + i + j - q_start[r];
      if (page_at != pos >> p.shift) {
        page_at = pos >> p.shift;
        g = page_of(r, page_at, len);
      }
      s[j] = g * p.page + (pos & (p.page - 1));
    }
    // (each part of the plan begins on a 16-byte boundary and is as long as whole pieces)
    *reinterpret_cast<int4*>(slot + i) = make_int4(s[0], s[1], s[2], s[3]);
    *reinterpret_cast<int4*>(request + i) = make_int4(o[0], o[1], o[2], o[3]);
  }
  // (other threads begin here than there: a small step's loads are then all on their way at once)
  for (int i = (i0 + step - step / 4) % step; i < n_pages; i += step) {
    const int r = find(new_base, p.requests, i);
    const int f = q_start[r + 1] - q_start[r], first = pages_of(kv_len[r] - f, p.shift), b = first + i - new_base[r];
    p.table[(size_t)r * p.table_ld + b] = page_of(r, b, kv_len[r] - f);
  }
  for (int i = (i0 + step / 2) % step; i < n_runs; i += step) {
    const int r = find(run_base, p.requests, i);
    const int f = q_start[r + 1] - q_start[r], len = kv_len[r] - f, b = (len >> p.shift) + i - run_base[r];
    const int from = max(len, b * p.page), to = (int)min((long long)kv_len[r], (long long)(b + 1) * p.page);
    reinterpret_cast<int4*>(p.buf + p.lay.runs)[i] =
        make_int4(q_start[r] + from - len, to - from, page_of(r, b, len), from - b * p.page);
  }
}

constexpr int kHeld = 1536;  // requests whose sums fit the block's shared memory

__global__ void __launch_bounds__(1024) k_plan(const PlanDev p) {
  __shared__ Sums warp_sum[32];
  __shared__ Sums carry_s;
  __shared__ int bad_s;
  __shared__ int held[6][kHeld + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5, n = p.requests;
  pdl_wait();
  pdl_launch();
  PlanHead* const head = reinterpret_cast<PlanHead*>(p.buf);
  int* const q_start = n <= kHeld ? held[0] : p.buf + p.lay.q_start;
  int* const new_base = n <= kHeld ? held[1] : p.buf + p.lay.new_base;
  int* const run_base = n <= kHeld ? held[2] : p.buf + p.lay.run_base;
  int* const tile_base = n <= kHeld ? held[4] : p.buf + p.lay.tile_base;
  int* const seg_base = n <= kHeld ? held[5] : p.buf + p.lay.seg_base;
  int* const kv_len = n <= kHeld ? held[3] : p.buf + p.lay.kv_len;
  const int free_n = p.free_pages ? *p.free_count : 0;
  // the page that is taken as the tid-th, if as many are: it comes while the sums are made
  const int nth = p.free_pages && free_n <= p.pages && tid < free_n ? p.free_pages[free_n - 1 - tid] : 0;
  bool odd = false;  // a page that the cache does not have
  if (tid == 0) {
    bad_s = 0;
    carry_s = Sums{0, 0, 0, 0, 0};
  }
  __syncthreads();
  // the sums, and whether the step can be had at all: a plan is made whole or not at all
  Sums total;
  for (int r0 = 0; r0 < n; r0 += blockDim.x) {
    const int r = r0 + tid;
    Sums mine{0, 0, 0, 0};
    int f = 0, len = 0, begun = 0;
    if (r < n) {
      f = p.fresh[r];
      len = p.length[r];
      if (p.free_pages && f > 0 && len > 0 && (len & (p.page - 1)) && (len >> p.shift) < p.max_blocks)
        begun = p.table[(size_t)r * p.table_ld + (len >> p.shift)];  // the page that its rows begin in
      if (!of_request(p, f, len, mine)) bad_s = 1;
    }
    Sums inc = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const Sums o = shfl_up(inc, d);
      if (lane >= d) inc = add(inc, o);
    }
    if (lane == 31) warp_sum[warp] = inc;
    __syncthreads();
    if (warp == 0) {
      Sums w = lane < warps ? warp_sum[lane] : Sums{0, 0, 0, 0, 0};
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const Sums o = shfl_up(w, d);
        if (lane >= d) w = add(w, o);
      }
      warp_sum[lane] = w;
    }
    __syncthreads();
    Sums base = carry_s;
    if (warp) base = add(base, warp_sum[warp - 1]);
    if (r < n) {
      q_start[r] = (int)min(base.rows + inc.rows - mine.rows, 0x7fffffffLL);
      new_base[r] = (int)min(base.pages + inc.pages - mine.pages, 0x7fffffffLL);
      run_base[r] = (int)min(base.runs + inc.runs - mine.runs, 0x7fffffffLL);
      tile_base[r] = (int)min(base.tiles + inc.tiles - mine.tiles, 0x7fffffffLL);
      seg_base[r] = (int)min(base.segs + inc.segs - mine.segs, 0x7fffffffLL);
      kv_len[r] = p.free_pages ? len + f : len;
    }
    odd |= (unsigned)begun >= (unsigned)p.pages;
    __syncthreads();
    if (tid == 0) carry_s = add(carry_s, warp_sum[warps - 1]);
    __syncthreads();
  }
  total = carry_s;
  int status = T2W_OK;
  // a call with little for a worker to do has no empty places: its shares are short, and every start counts the same
  const int extra = total.tiles >= 8LL * p.cut.workers ? p.cut.extra : 0;
  total.tiles += extra * total.segs;
  if (bad_s || total.rows > p.rows || total.tiles > 0x7fffffffLL) status = T2W_ERR_INVALID;
  else if (p.free_pages && (free_n < 0 || free_n > p.pages)) status = T2W_ERR_INVALID;
  else if (p.free_pages && total.pages > free_n) status = T2W_ERR_EXHAUSTED;
  if (status == T2W_OK) {  // (for all threads alike)
    auto no_page = [&](int g) { return (unsigned)g >= (unsigned)p.pages; };
    odd |= tid < total.pages && no_page(nth);
    const int more = (int)total.pages - (int)blockDim.x;  // the first `more` entries from lo on: four at a time, but for the ends
    if (more > 0) {
      const int* const lo = p.free_pages + free_n - (int)total.pages;
      const int head = min(more, (int)(-(reinterpret_cast<intptr_t>(lo) >> 2) & 3)), fours = (more - head) / 4;
      if (tid < head) odd |= no_page(lo[tid]);
      if (tid < more - head - 4 * fours) odd |= no_page(lo[head + 4 * fours + tid]);
#pragma unroll 4
      for (int i = tid; i < fours; i += blockDim.x) {
        const int4 g = reinterpret_cast<const int4*>(lo + head)[i];
        odd |= no_page(g.x) | no_page(g.y) | no_page(g.z) | no_page(g.w);
      }
    }
    if (__syncthreads_or(odd)) status = T2W_ERR_INVALID;
  }
  __syncthreads();
  if (status != T2W_OK) {  // void: no rows, no pages, the lengths as they were
    total = Sums{0, 0, 0, 0, 0};
    for (int r = tid; r < n; r += blockDim.x) {
      q_start[r] = new_base[r] = run_base[r] = tile_base[r] = seg_base[r] = 0;
      kv_len[r] = p.length[r];
    }
  }
  if (extra)
    for (int r = tid; r < n; r += blockDim.x) tile_base[r] += extra * seg_base[r];
  const int n_rows = (int)total.rows, n_pages = (int)total.pages, n_runs = (int)total.runs, tiles = (int)total.tiles;
  const int per = max((int)(((long long)tiles + p.cut.workers - 1) / p.cut.workers), p.cut.min_per);
  const int workers = tiles ? (int)(((long long)tiles + per - 1) / per) : 0;
  if (tid == 0) {
    q_start[n] = n_rows;
    new_base[n] = n_pages;
    run_base[n] = n_runs;
    tile_base[n] = tiles;
    *head = PlanHead{n_runs, tiles, per, workers, status, n_rows, free_n - n_pages, extra};
  }
  __syncthreads();
  if (n <= kHeld) {
    for (int r = tid; r <= n; r += blockDim.x) {
      p.buf[p.lay.q_start + r] = q_start[r];
      p.buf[p.lay.new_base + r] = new_base[r];
      p.buf[p.lay.run_base + r] = run_base[r];
      if (r < n) p.buf[p.lay.kv_len + r] = kv_len[r];
    }
  }
  // the workers' starts: worker w begins at tile w * per of all
  for (int w = tid; w < workers; w += blockDim.x) {
    const int r = find(tile_base, n, w * per);
    const int f = q_start[r + 1] - q_start[r], kv = kv_len[r], nq = (f + p.cut.tq - 1) / p.cut.tq;
    const int one = (tile_base[r + 1] - tile_base[r]) / p.kv_heads;  // places of one key head
    const int rem = w * per - tile_base[r], hk = rem / one, in = rem - hk * one;
    auto before = [&](int x) { return (int)tiles_before(f, kv, p.causal, p.cut.tq, p.cut.kt, x) + x * extra; };
    int lo = 0, hi = nq;  // the query tile: the last x with before(x) <= in
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before(mid) <= in) lo = mid; else hi = mid;
    }
    int place = w * per, kt = in - before(lo) - extra, seg_r = r, seg_h = hk, seg_q = lo, row0 = q_start[r], rows = f, keys = kv;
    const int nt = seg_tiles(tile_keys(f, kv, p.causal, p.cut.tq, lo), p.cut.kt);
    if (p.cut.whole && kt > -extra && 5 * (nt + extra) <= 3 * per) {  // a short segment is not cut
      if (2 * kt < nt) {
        place -= kt + extra;
      } else {  // the next one begins the share
        place += nt - kt;
        if (++seg_q == nq) {
          seg_q = 0;
          if (++seg_h == p.kv_heads) {
            seg_h = 0;
            do ++seg_r;
            while (seg_r < n && q_start[seg_r + 1] == q_start[seg_r]);
            if (seg_r < n) {
              row0 = q_start[seg_r];
              rows = q_start[seg_r + 1] - row0;
              keys = kv_len[seg_r];
            }
          }
        }
      }
      kt = -extra;
    }
    // request, key head, query tile and key tile (below 0 where the share begins with empty places); then what a worker
    // would look up for that request, and the share's first place
    int4* const start = reinterpret_cast<int4*>(p.buf + p.lay.starts) + 2 * w;
    start[0] = make_int4(seg_r, seg_h, seg_q, kt);
    start[1] = make_int4(row0, rows, keys, place);
  }
  if (tid == 0) {  // where the last share ends
    int4* const start = reinterpret_cast<int4*>(p.buf + p.lay.starts) + 2 * workers;
    start[0] = make_int4(0, 0, 0, 0);
    start[1] = make_int4(0, 0, 0, tiles);
  }
  if (!p.scattered)
    scatter(p, q_start, new_base, run_base, kv_len, n_rows, n_pages, n_runs, free_n, tid, blockDim.x);
  // where the caller keeps its lengths: last, since they may be what was read above
  if (p.kv_len_out)
    for (int r = tid; r < n; r += blockDim.x) p.kv_len_out[r] = kv_len[r];
  if (p.free_left_out && tid == 0) *p.free_left_out = free_n - n_pages;
}

// The second launch of a large step.
__global__ void __launch_bounds__(256) k_plan_rows(const PlanDev p) {
  pdl_wait();
  pdl_launch();
  __shared__ int held[4][kHeld + 1];
  const PlanHead h = *reinterpret_cast<const PlanHead*>(p.buf);
  const int n = p.requests, n_pages = p.buf[p.lay.new_base + n];
  const int *q_start = p.buf + p.lay.q_start, *new_base = p.buf + p.lay.new_base, *run_base = p.buf + p.lay.run_base,
            *kv_len = p.buf + p.lay.kv_len;
  if (n <= kHeld) {
    for (int r = threadIdx.x; r <= n; r += blockDim.x) {
      held[0][r] = q_start[r];
      held[1][r] = new_base[r];
      held[2][r] = run_base[r];
      if (r < n) held[3][r] = kv_len[r];
    }
    __syncthreads();
    q_start = held[0];
    new_base = held[1];
    run_base = held[2];
    kv_len = held[3];
  }
  scatter(p, q_start, new_base, run_base, kv_len, h.used, n_pages, h.n_runs, h.free_left + n_pages,
          blockIdx.x * blockDim.x + threadIdx.x, gridDim.x * blockDim.x);
}

// Pages of finished requests back onto the end of the free list, in request and block order; their lengths become 0.  All
// of it is looked at before any of it is written, so that a release is made whole or not at all.  The block takes up to 4096
// requests at a time, four a thread; their pages are then dealt to the threads four in a row, which find their request by a
// search in the sums: one long request's pages are spread over all threads like those of many.  Measured, on the GPU: 4
// requests of 400 tokens in pages of 16 take 8 us, 64 of 2000 15, one of 150 thousand 14, 3000 of 100 33.
constexpr int kReleaseThreads = 1024, kReleaseAtOnce = 4 * kReleaseThreads;
__global__ void __launch_bounds__(kReleaseThreads) k_release(const int* done, int* length, int* table, int n, int shift,
                                                             int table_ld, int max_blocks, int pages, int* free_pages,
                                                             int* free_count, int* status) {
  __shared__ long long warp_sum[32];
  __shared__ int base[kReleaseAtOnce];  // pages of the requests before
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_launch();
  const int at0 = *free_count;
  // The pages that requests r0 .. give back (base), and how many they are together; -1 where a length cannot be.
  auto sums = [&](int r0) -> long long {
    int mine[4], ends[4], lens[4];
    bool bad = false;
    long long inc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = r0 + 4 * tid + j;
      ends[j] = r < n ? done[r] : 0;
      lens[j] = r < n ? length[r] : 0;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool fits = lens[j] >= 0 && pages_of(lens[j], shift) <= max_blocks;
      bad |= ends[j] && !fits;
      mine[j] = ends[j] && fits ? pages_of(lens[j], shift) : 0;
      inc += mine[j];
    }
    long long before = -inc;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long o = __shfl_up_sync(~0u, inc, d);
      if (lane >= d) inc += o;
    }
    if (lane == 31) warp_sum[warp] = inc;
    bad = __syncthreads_or(bad);
    if (warp == 0) {
      long long w = warp_sum[lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(~0u, w, d);
        if (lane >= d) w += o;
      }
      warp_sum[lane] = w;
    }
    __syncthreads();
    before += inc + (warp ? warp_sum[warp - 1] : 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      base[4 * tid + j] = (int)min(before, 0x7fffffffLL);
      before += mine[j];
    }
    const long long sum = warp_sum[kReleaseThreads / 32 - 1];
    __syncthreads();
    return bad ? -1 : sum;
  };
  // Pages i0 .. i0 + 3 of those (the last one again where there are fewer).
  auto entries = [&](int r0, int i0, int sum, int* (&at)[4], int (&e)[4]) {
    const int m = min(kReleaseAtOnce, n - r0);
    int r = find(base, m, i0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = min(i0 + j, sum - 1);
      if (r + 1 < m && base[r + 1] <= i) {  // mostly the next one's
        ++r;
        if (r + 1 < m && base[r + 1] <= i) r = find(base, m, i);
      }
      at[j] = table + (size_t)(r0 + r) * table_ld + i - base[r];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = *at[j];
  };
  int* from[4];
  int e[4];
  bool bad = at0 < 0 || at0 > pages;
  long long at = at0, sum = 0;
  for (int r0 = 0; r0 < n && !bad; r0 += kReleaseAtOnce) {
    sum = sums(r0);
    at += sum;
    bool odd = sum < 0 || at > pages;  // more pages than there are: one of them was given back before
    if (!odd)
      for (long long i = 4 * tid; i < sum; i += 4 * kReleaseThreads) {
        entries(r0, (int)i, (int)sum, from, e);
#pragma unroll
        for (int j = 0; j < 4; ++j) odd |= (unsigned)e[j] >= (unsigned)pages;
      }
    bad = __syncthreads_or(odd);
  }
  if (bad) {
    if (tid == 0) atomicExch(status, T2W_ERR_INVALID);
    return;
  }
  at = at0;
  for (int r0 = 0; r0 < n; r0 += kReleaseAtOnce) {
    if (n > kReleaseAtOnce) sum = sums(r0);  // (of one turn they are there)
    for (long long i = 4 * tid; i < sum; i += 4 * kReleaseThreads) {
      entries(r0, (int)i, (int)sum, from, e);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < sum) {
          free_pages[at + i + j] = e[j];
          *from[j] = -1;
        }
    }
    for (int r = r0 + tid; r < min(n, r0 + kReleaseAtOnce); r += kReleaseThreads)
      if (done[r]) length[r] = 0;
    at += sum;
    __syncthreads();
  }
  if (tid == 0) *free_count = (int)at;
}

bool page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }
int page_shift(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

}  // namespace
}  // namespace t2w

using namespace t2w;

extern "C" int64_t t2w_paged_plan_ints(int32_t requests, int32_t rows, int32_t max_fresh, int32_t page, int32_t q_heads,
                                       int32_t kv_heads, int32_t head_dim, int64_t* at) {
  if (requests <= 0 || rows < 0 || max_fresh <= 0 || !page_ok(page) || kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads)
    return T2W_ERR_INVALID;
  if ((head_dim != 64 && head_dim != 128) || q_heads / kv_heads > 128) return T2W_ERR_UNSUPPORTED;
  const PlanLayout l = paged_layout(requests, rows, page, paged_cut(max_fresh, q_heads, kv_heads, head_dim));
  if (l.total > 0x7fffffffLL) return T2W_ERR_INVALID;
  if (at) {
    at[0] = l.q_start;
    at[1] = l.kv_len;
    at[2] = l.slot;
    at[3] = l.request;
  }
  return l.total;
}

extern "C" int t2w_paged_plan(const t2w_paged_plan_args* a, void* stream) {
  if (!a || !a->fresh || !a->length || !a->table || !a->plan || (reinterpret_cast<uintptr_t>(a->plan) & 15))
    return T2W_ERR_INVALID;
  if ((a->free_pages == nullptr) != (a->free_count == nullptr)) return T2W_ERR_INVALID;
  if (a->max_blocks <= 0 || a->table_ld < a->max_blocks || a->pages <= 0 || (int64_t)a->pages * a->page > 0x7fffffffLL)
    return T2W_ERR_INVALID;
  const int64_t ints = t2w_paged_plan_ints(a->requests, a->rows, a->max_fresh, a->page, a->q_heads, a->kv_heads,
                                           a->head_dim, nullptr);
  if (ints < 0) return (int)ints;
  PlanDev p;
  p.requests = a->requests;
  p.rows = a->rows;
  p.max_fresh = a->max_fresh;
  p.page = a->page;
  p.shift = page_shift(a->page);
  p.table_ld = a->table_ld;
  p.max_blocks = a->max_blocks;
  p.pages = a->pages;
  p.causal = a->causal != 0;
  p.kv_heads = a->kv_heads;
  p.cut = paged_cut(a->max_fresh, a->q_heads, a->kv_heads, a->head_dim);
  p.lay = paged_layout(a->requests, a->rows, a->page, p.cut);
  p.fresh = a->fresh;
  p.length = a->length;
  p.table = a->table;
  p.free_pages = a->free_pages;
  p.free_count = a->free_count;
  p.kv_len_out = a->kv_len;
  p.free_left_out = a->free_left;
  p.buf = a->plan;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  p.scattered = a->rows > 4096;
  const bool small = a->rows <= 1024 && a->requests <= 256;
  cudaError_t e = launch_k(k_plan, dim3(1), dim3(small ? 512 : 1024), 0, st, p);
  if (e == cudaSuccess && p.scattered) {
    const int grid = (a->rows + 1023) / 1024;
    e = launch_k(k_plan_rows, dim3(grid < 2 * num_sms() ? grid : 2 * num_sms()), dim3(256), 0, st, p);
  }
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return T2W_ERR_CUDA;
  }
  return T2W_OK;
}

extern "C" int t2w_paged_status(const int32_t* plan, void* stream) {
  if (!plan) return T2W_ERR_INVALID;
  int32_t v = 0;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(&v, &reinterpret_cast<const PlanHead*>(plan)->status, sizeof v, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return T2W_ERR_CUDA;
  }
  return v;
}

extern "C" int t2w_paged_release(const int32_t* done, int32_t* length, int32_t* table, int32_t requests, int32_t page,
                                 int32_t table_ld, int32_t max_blocks, int32_t pages, int32_t* free_pages,
                                 int32_t* free_count, int32_t* status, void* stream) {
  if (!done || !length || !table || !free_pages || !free_count || !status || requests <= 0 || !page_ok(page) ||
      max_blocks <= 0 || table_ld < max_blocks || pages <= 0)
    return T2W_ERR_INVALID;
  const cudaError_t e = launch_k(k_release, dim3(1), dim3(kReleaseThreads), 0, static_cast<cudaStream_t>(stream),
                                 done, length, table, requests, page_shift(page), table_ld, max_blocks, pages, free_pages, free_count,
                                 status);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return T2W_ERR_CUDA;
  }
  return T2W_OK;
}
