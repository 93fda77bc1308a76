// Pages of a step in which rows go on from other rows, are cut, or end.
//
// Row i takes over the first n_i = min(keep_i, len of its parent) tokens: n_i / P whole pages, which any number of rows may hold together since nothing
// is written into a whole page any more, and a begun one of n_i % P tokens.  A begun page stays with one row: none where some row holds it
// whole, else a row that goes on from itself, else the lowest.  The others take a new page each, in the order of the rows, and an entry {page, new
// page, n_i % P} of the list of copies.  Pages that rows held before and none holds any more go back on top of the free list, in
// ascending order: the taken ones stand in front of free_head, so there is room for them.
//
// No count of a page's holders is kept: one word a page takes the minimum of what the rows say of it (0 held whole, 1 + key begun, AE_HELD
// held before; AE_UNUSED none of these), so the order of the atomics does not show in the result.
// Expects AE_LIST_ROWS (most rows), AE_LIST_THREADS, AE_LIST_CTAS, AE_LIST_BATCH (table entries of a thread on their way together).
#define AE_HELD 0xfffffffeu
#define AE_UNUSED 0xffffffffu

struct AeForkSmem {
  int parent[AE_LIST_ROWS];  // -1: the row ends
  int n[AE_LIST_ROWS];       // tokens of it
  int last[AE_LIST_ROWS];    // its begun page; -1: none
  int held[AE_LIST_ROWS];    // pages that the row held before
  int warp_sum[3][AE_LIST_THREADS / 32];
  u32 bad;
};

extern "C" __global__ void __launch_bounds__(AE_LIST_THREADS) ae_plan_forks(const __grid_constant__ AePlanForksArgs a) {
  extern __shared__ u8 smem_raw[];
  AeForkSmem& sm = *(AeForkSmem*)smem_raw;
  ae_grid_wait();
  ae_grid_trigger();
  const int cta = (int)cluster_ctarank(), tid = (int)threadIdx.x, lane = tid & 31;
  const int gtid = cta * AE_LIST_THREADS + tid, gstep = AE_LIST_CTAS * AE_LIST_THREADS;
  const int P = 1 << a.page_log2, B = a.B, W = a.max_pages;
  const i64 most = (i64)W << a.page_log2;  // tokens that a row of the table holds
  u32 bad = 0;
  if (tid == 0) sm.bad = 0;
  // what is on the free list before: a head outside of it is cut
  const int head = min(max(*a.free_head, 0), a.n_free);

  // phase 0: the pages' words, and every CTA for itself what the rows take over
  const int groups = (a.num_pages + 3) / 4;
  if (gtid == 0) *a.status = 0;
  for (int i = gtid; i < groups; i += gstep) ((uint4*)a.state)[i] = make_uint4(AE_UNUSED, AE_UNUSED, AE_UNUSED, AE_UNUSED);
  auto len_of = [&](int r, u32& flags) {
    const int n = a.lens[r];
    if (n < 0) flags |= 8u;
    if (n > most) flags |= 2u;
    return (int)min((i64)max(n, 0), most);
  };
  for (int r = tid; r < B; r += AE_LIST_THREADS) {
    int p = a.parents[r], n = 0, last = -1;
    sm.held[r] = (int)(((i64)len_of(r, bad) + P - 1) >> a.page_log2);
    const int keep = a.keep ? a.keep[r] : 0;
    if (p < -1 || p >= B) {
      bad |= 8u;
      p = -1;
    }
    if (p >= 0) {
      n = len_of(p, bad);
      if (a.keep) {
        if (keep < 0 || keep > n) bad |= 8u;
        n = min(max(keep, 0), n);
      }
      if (n & (P - 1)) last = a.table[(i64)p * a.table_stride + (n >> a.page_log2)];
      if (last < 0 || last >= a.num_pages) {
        if (n & (P - 1)) {  // a page outside the pool holds nothing
          bad |= 16u;
          n &= ~(P - 1);
        }
        last = -1;
      }
    }
    sm.parent[r] = p;
    sm.n[r] = n;
    sm.last[r] = last;
  }
  ae_phase_end();

  // phase 1: what the rows say of the pages; the whole pages of the new table
  for (int r = gtid; r < B; r += gstep)
    if (sm.last[r] >= 0) atomicMin(a.state + sm.last[r], 1u + (u32)r + (sm.parent[r] == r ? 0u : (u32)B));
  const int warps = gstep / 32, chunks = (W + 31) / 32;
  const int gwarp = cta * (AE_LIST_THREADS / 32) + (tid >> 5);
  for (int i0 = gwarp; i0 < B * chunks; i0 += warps * AE_LIST_BATCH) {
    int before[AE_LIST_BATCH], now[AE_LIST_BATCH];
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {  // the reads in front of the atomics, which the compiler moves no read across
      before[j] = now[j] = 0;
      const int i = min(i0 + j * warps, B * chunks - 1), r = i / chunks, c = (i - r * chunks) * 32 + lane;
      const int p = sm.parent[r], whole = sm.n[r] >> a.page_log2;
      if (c < sm.held[r]) before[j] = a.table[(i64)r * a.table_stride + c];
      if (c < whole) now[j] = a.table[(i64)p * a.table_stride + c];
    }
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      const int i = i0 + j * warps;
      if (i >= B * chunks) break;
      const int r = i / chunks, c = (i - r * chunks) * 32 + lane, whole = sm.n[r] >> a.page_log2;
      if (c < sm.held[r]) {
        if (before[j] >= 0 && before[j] < a.num_pages)
          atomicMin(a.state + before[j], AE_HELD);
        else
          bad |= 16u;
      }
      if (c < whole && now[j] >= 0 && now[j] < a.num_pages) atomicMin(a.state + now[j], 0u);
      if (c < W && (c != whole || sm.last[r] < 0)) a.table_out[(i64)r * W + c] = now[j];
    }
  }
  ae_phase_end();

  // phase 2: which rows copy (every CTA all of them, 8 rows a thread at most), and the pages that nobody holds any more
  const int per = (B + AE_LIST_THREADS - 1) / AE_LIST_THREADS, r0 = min(tid * per, B), r1 = min(r0 + per, B);
  u32 copy = 0;  // of row r0 + j: bit j
  for (int r = r0; r < r1; ++r)
    if (sm.last[r] >= 0 && __ldcg(a.state + sm.last[r]) != 1u + (u32)r + (sm.parent[r] == r ? 0u : (u32)B)) copy |= 1u << (r - r0);
  int taken, order = ae_cta_scan(__popc(copy), sm.warp_sum[0], taken);
  int first, end, freed = 0;
  ae_page_share(a.num_pages, cta, first, end);
  const int share = (end - first) / 4, tper = (share + AE_LIST_THREADS - 1) / AE_LIST_THREADS;
  const int g0 = first / 4 + min(tid * tper, share), g1 = min(g0 + tper, end / 4);
#pragma unroll 4
  for (int g = g0; g < g1; ++g) {
    const uint4 u = __ldcg((const uint4*)a.state + g);
    freed += (u.x == AE_HELD) + (u.y == AE_HELD) + (u.z == AE_HELD) + (u.w == AE_HELD);
  }
  int cta_freed;
  int before = ae_cta_scan(freed, sm.warp_sum[1], cta_freed);
  if (tid == 0) a.counts[cta] = cta_freed;
  if (bad) atomicOr(&sm.bad, bad);
  ae_phase_end();

  // phase 3: the lists
  int all_freed = 0;
#pragma unroll
  for (int i = 0; i < AE_LIST_CTAS; ++i) {
    const int n = __ldcg(a.counts + i);
    if (i < cta) before += n;
    all_freed += n;
  }
  const int got = min(taken, a.n_free - head), top = max(head + got - all_freed, 0);
  // page j of those freed stands at top + j, as far as there is room
  const int room = head + got - top;
  for (int g = g0; g < g1 && freed > 0; ++g) {
    const uint4 u = __ldcg((const uint4*)a.state + g);
    const u32 w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (w[k] == AE_HELD) {
        if (before < room) a.free_out[top + before] = g * 4 + k;
        ++before;
      }
  }
  for (int i = gtid; i < a.n_free; i += gstep)
    if (i < top || i >= top + min(room, all_freed)) a.free_out[i] = a.free_pages[i];
  u32 late = 0;
  for (int r = r0; r < r1; ++r) {  // every CTA a share of the rows, for the writes
    const bool copies = copy >> (r - r0) & 1;
    const int mine = order;
    order += copies;
    if (r % AE_LIST_CTAS != cta) continue;
    int n = sm.n[r];
    const int part = n & (P - 1);
    if (sm.last[r] >= 0) {
      int page = sm.last[r];
      if (copies) {
        page = head + mine < a.n_free ? a.free_pages[head + mine] : -1;
        if (head + mine >= a.n_free) late |= 1u;
        if (page >= a.num_pages || (page < 0 && head + mine < a.n_free)) late |= 16u;
        AePageCopy e = {sm.last[r], page, part, 0};
        if (page < 0 || page >= a.num_pages) {  // no page: the row ends with its whole ones
          n -= part;
          page = 0;
          // the list ends where the free pages did; a page outside the pool leaves no gap in it
          e.dst = e.src;
          if (head + mine >= a.n_free) e.src = e.dst = e.slots = 0;
        }
        a.copies[mine] = e;
      }
      a.table_out[(i64)r * W + (sm.n[r] >> a.page_log2)] = page;
    }
    a.lens_out[r] = n;
  }
  for (int i = gtid; i < B; i += gstep)
    if (i >= taken) {
      const AePageCopy none = {0, 0, 0, 0};
      a.copies[i] = none;
    }
  if (all_freed > room) late |= 4u;
  if (tid == 0) late |= sm.bad;
  if (late) atomicOr(a.status, late);
  if (gtid == 0) *a.head_out = top;
}
