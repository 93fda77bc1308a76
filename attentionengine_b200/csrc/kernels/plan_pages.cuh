// Pages of one step of a serving loop, from the rows' lengths: which free pages the rows take, the slot and position of every new
// token, and the segments (runs of new tokens inside one page) that the write into the cache works on.
//
// With P slots a page, have = ceil(old / P) and want = ceil((old + new) / P), row b takes want - have pages, the i-th of them
// free_pages[head + sum of the earlier rows' needs + i].  Everything else is arithmetic on three running sums over the rows (new
// tokens, needed pages, segments), so every CTA makes the sums for itself (at most 4096 rows: 16 a thread, two block scans) and then
// takes its share of the tokens, pages and segments; each finds its row by bisection in shared memory.  One launch, no CTA waits for another,
// and what a CTA writes into the table no CTA reads: entries below `have` are read, new ones are looked up in free_pages.
// Latency-bound.
// Bits of the status word: 1 free pages ran out, 2 a row outgrew the table, 4 more new tokens than n_tokens (the later ones are left out),
// 8 a negative length (taken as 0).  A token without a page has slot -1 and its segment no tokens.
// Expects AE_PLAN_ROWS (most rows).

#define AE_PLAN_THREADS 256

struct AePlanSmem {
  int cu[AE_PLAN_ROWS + 1];     // first new token of each row
  int take[AE_PLAN_ROWS + 1];   // first needed page
  int seg[AE_PLAN_ROWS + 1];    // first segment
  i64 warp_sum[2][AE_PLAN_THREADS / 32];
  u32 bad;
};

// Exclusive sum over the block; `total` is the whole.
AE_DEVICE i64 ae_block_scan(i64 x, i64* warp_sum, i64& total) {
  const u32 lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  i64 s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const i64 y = __shfl_up_sync(0xffffffffu, s, o);
    if ((int)lane >= o) s += y;
  }
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  i64 before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < AE_PLAN_THREADS / 32; ++w) {
    if (w < (int)warp) before += warp_sum[w];
    total += warp_sum[w];
  }
  return before + s - x;
}

// The row whose share of a running sum holds item i: the last r with first[r] <= i (rows without a share are passed over).
AE_DEVICE int ae_row_of(const int* first, int B, int i) {
  int lo = 0, hi = B;  // first[lo] <= i < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= i)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

extern "C" __global__ void __launch_bounds__(AE_PLAN_THREADS) ae_plan_pages(const __grid_constant__ AePlanPagesArgs a) {
  extern __shared__ u8 smem_raw[];
  AePlanSmem& sm = *(AePlanSmem*)smem_raw;
  ae_grid_wait();  // brought up under the kernel in front
  ae_grid_trigger();
  const int P = 1 << a.page_log2;
  const int per = (a.B + AE_PLAN_THREADS - 1) / AE_PLAN_THREADS;  // rows of a thread
  const int r0 = min((int)threadIdx.x * per, a.B), r1 = min(r0 + per, a.B);
  const i64 head = max(*a.free_head, 0);
  u32 bad = 0;
  auto old_len = [&](int r) { return max(a.old_lens[r], 0); };
  if (threadIdx.x == 0) sm.bad = 0;

  i64 sum = 0, total;
  for (int r = r0; r < r1; ++r) {
    const int n = a.new_lens[r];
    if (n < 0 || a.old_lens[r] < 0) bad |= 8u;
    sum += max(n, 0);
  }
  const i64 first = ae_block_scan(sum, sm.warp_sum[0], total);
  if (total > a.n_tokens) bad |= 4u;
  // pages from `have` to `want`, segments: pages of the table that get a token
  auto pages = [&](int r, i64 n, int& need, int& n_seg, bool& outgrown) {
    const i64 o = old_len(r);
    const i64 h = (o + P - 1) >> a.page_log2, w = (o + n + P - 1) >> a.page_log2;
    need = (int)(min(w, (i64)a.max_pages) - min(h, (i64)a.max_pages));
    outgrown = w > a.max_pages;
    n_seg = n > 0 ? (int)(w - (o >> a.page_log2)) : 0;
  };
  i64 at = first, mine = 0, all;  // needed pages, and segments above them
  for (int r = r0; r < r1; ++r) {
    const i64 from = min(at, (i64)a.n_tokens);
    at += max(a.new_lens[r], 0);
    sm.cu[r] = (int)from;
    int need, n_seg;
    bool outgrown;
    pages(r, min(at, (i64)a.n_tokens) - from, need, n_seg, outgrown);
    mine += (i64)n_seg << 32 | (u32)need;
    if (outgrown) bad |= 2u;
  }
  mine = ae_block_scan(mine, sm.warp_sum[1], all);
  at = first;
  for (int r = r0; r < r1; ++r) {
    const i64 from = min(at, (i64)a.n_tokens);
    at += max(a.new_lens[r], 0);
    int need, n_seg;
    bool outgrown;
    pages(r, min(at, (i64)a.n_tokens) - from, need, n_seg, outgrown);
    sm.take[r] = (int)(u32)mine;
    sm.seg[r] = (int)(mine >> 32);
    mine += (i64)n_seg << 32 | (u32)need;
  }
  const int all_need = (int)(u32)all, all_segs = (int)(all >> 32);
  if (threadIdx.x == 0) {
    sm.cu[a.B] = (int)min(total, (i64)a.n_tokens);
    sm.take[a.B] = all_need;
    sm.seg[a.B] = all_segs;
    if (head + all_need > a.n_free) bad |= 1u;
  }
  if (bad) atomicOr(&sm.bad, bad);
  __syncthreads();

  // page i of row r, which may be one that this step takes
  auto page_of = [&](int r, i64 i) -> int {
    if (i >= a.max_pages) return -1;
    const int have = (int)min((i64)((old_len(r) + (i64)P - 1) >> a.page_log2), (i64)a.max_pages);
    if (i < have) return a.table[(i64)r * a.table_stride + i];
    const i64 f = head + sm.take[r] + (i - have);
    return f < a.n_free ? a.free_pages[f] : -1;
  };
  const int tid = (int)(blockIdx.x * AE_PLAN_THREADS + threadIdx.x), step = (int)(gridDim.x * AE_PLAN_THREADS);
  // Token, segment, needed page and row i of all: their table and free-page reads are on their way together (one after the other, four
  // loops took 1 us more of a step of 256 rows).
  const int n_tok = sm.cu[a.B], most = max(max(a.n_tokens, a.n_seg), max(all_need, a.B + 1));
  for (int i = tid; i < most; i += step) {
    int page_t = -1, page_s = -1, page_n = -1, row_s = 0, row_n = 0, into = 0, j = 0;
    i64 pos = -1;
    if (i < n_tok) {
      const int r = ae_row_of(sm.cu, a.B, i);
      pos = (i64)old_len(r) + (i - sm.cu[r]);
      page_t = page_of(r, pos >> a.page_log2);
    }
    if (i < all_segs) {
      row_s = ae_row_of(sm.seg, a.B, i);
      j = i - sm.seg[row_s];
      const i64 o = old_len(row_s);
      into = (int)(o & (P - 1));
      page_s = page_of(row_s, (o >> a.page_log2) + j);
    }
    if (i < all_need) {
      row_n = ae_row_of(sm.take, a.B, i);
      if (head + i < a.n_free) page_n = a.free_pages[head + i];
    }
    if (i < a.n_tokens) {
      a.positions[i] = (int)pos;
      a.slots[i] = page_t < 0 ? -1 : ((i64)page_t << a.page_log2) + (pos & (P - 1));
    }
    if (i < a.n_seg) {
      AePageSegment e = {0, 0, 0, 0};
      if (page_s >= 0) {
        e.page = page_s;
        e.slot = j == 0 ? into : 0;
        e.token = sm.cu[row_s] + (j == 0 ? 0 : j * P - into);
        e.tokens = min(sm.cu[row_s + 1], e.token + P - e.slot) - e.token;
      }
      a.segments[i] = e;
    }
    if (i < all_need) {
      const int have = (int)min((i64)((old_len(row_n) + (i64)P - 1) >> a.page_log2), (i64)a.max_pages);
      a.table[(i64)row_n * a.table_stride + have + (i - sm.take[row_n])] = page_n;
    }
    if (i <= a.B) {
      a.cu[i] = sm.cu[i];
      if (i < a.B) a.lens[i] = old_len(i) + (sm.cu[i + 1] - sm.cu[i]);
    }
  }
  if (tid == 0) {
    *a.head_out = (int)min(head + all_need, (i64)a.n_free);
    *a.status = sm.bad;
  }
}
