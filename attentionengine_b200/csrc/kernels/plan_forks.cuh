// Pages of a step in which rows go on from other rows, are cut, or end.
//
// Row i takes over the first n_i = min(keep_i, len of its parent) tokens: n_i / P whole pages, which any number of rows may hold together since nothing
// is written into a whole page any more, and a begun one of n_i % P tokens.  A begun page stays with one row: none where some row holds it
// whole, else a row that goes on from itself, else the lowest.  The others take a new page each, in the order of the rows, and an entry {page, new
// page, n_i % P} of the list of copies.  New pages are the free list's; behind those, the ones that rows held before and none holds any more, in
// ascending order (none of them is read by a copy, since a copy's page is one that some row has begun).  The rest of the latter goes back on top of the free list, in
// ascending order: the taken ones stand in front of free_head, so there is room for them.
//
// No count of a page's holders is kept.  Phase 1 says what every row takes over and clears the bitmaps; phase 2 sets the pages' bits (held before, held
// whole, begun), finds the row that keeps a begun page as the minimum of a key, and writes the whole pages of the new table; phase 3 is a running
// sum over the rows that copy and one over the pages that are held no more.
#define AE_FORK_KEY(r, parent) ((u32)(r) + ((parent) == (r) ? 0u : (u32)a.B))

AE_DEVICE void ae_fork_rows(const AePlanForksArgs& a, const AeListState& st, const AeListShare sh) {
  if (sh.first() == 0) *a.status = 0;
  for (u32 i = sh.first(); i < 3u * (u32)a.words / 4; i += sh.step()) ((uint4*)st.held)[i] = make_uint4(0, 0, 0, 0);
  const i64 most = (i64)a.max_pages << a.page_log2;  // tokens that a row of the table holds
  const int P = 1 << a.page_log2;
  for (u32 i = sh.first(); i < (u32)a.B; i += sh.step()) {
    const int r = (int)i, len = a.lens[r], keep = a.keep ? a.keep[r] : 0x7fffffff;
    int p = a.parents[r], n = 0, last = -1;
    if (p < -1 || p >= a.B) p = -1;
    if (p >= 0) {
      n = min(max(keep, 0), (int)min((i64)max(a.lens[p], 0), most));
      if (n & (P - 1)) {
        last = a.table[(i64)p * a.table_stride + (n >> a.page_log2)];
        if (ae_in_pool(last, a.num_pages)) {
          st.owner[last] = 0xffffffffu;
        } else {  // a page outside the pool holds nothing
          n &= ~(P - 1);
          last = -1;
        }
      }
    }
    st.rows[r] = make_int4(p, n, last, (int)((min((i64)max(len, 0), most) + P - 1) >> a.page_log2));
  }
}

// What is wrong with a row's numbers; *status is cleared in the phase before.
AE_DEVICE u32 ae_fork_check(const AePlanForksArgs& a, const int4 row, int r) {
  const i64 most = (i64)a.max_pages << a.page_log2;
  const int len = a.lens[r], p = a.parents[r];
  u32 bad = len < 0 ? 8u : len > most ? 2u : 0u;
  if (p < -1 || p >= a.B) bad |= 8u;
  if (row.x >= 0) {
    const int had = (int)min((i64)max(a.lens[row.x], 0), most), want = a.keep ? a.keep[r] : had;
    if (want < 0 || want > had) bad |= 8u;
    if (row.y != min(max(want, 0), had)) bad |= 16u;  // its begun page was left out
  }
  return bad;
}

AE_DEVICE void ae_fork_marks(const AePlanForksArgs& a, const AeListState& st, const AeListShare sh) {
  u32 bad = 0;
  for (u32 r = sh.first(); r < (u32)a.B; r += sh.step()) {
    const int4 row = st.rows[r];
    bad |= ae_fork_check(a, row, (int)r);
    if (row.z >= 0) {
      ae_set_bit(st.begun, row.z);
      atomicMin(st.owner + row.z, AE_FORK_KEY((int)r, row.x));
    }
  }
  for (AeEntries e(sh, a.B, a.max_pages); e.more();) {
    int at[AE_LIST_BATCH], before[AE_LIST_BATCH], now[AE_LIST_BATCH];  // at: bit 0 held before, 1 whole now, 2 the row's own, 3 to be written
    const u32 i0 = e.i;
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {  // the reads in front of the atomics, which the compiler moves no read across
      at[j] = before[j] = now[j] = 0;
      if (e.more()) {
        const int4 row = st.rows[e.r];
        const int whole = row.y >> a.page_log2;
        at[j] = (e.c < row.w) | (e.c < whole) << 1 | (row.x == e.r) << 2 | (e.c != whole || row.z < 0) << 3;
        if (at[j] & 1) before[j] = a.table[(i64)e.r * a.table_stride + e.c];
        if ((at[j] & 6) == 2) now[j] = a.table[(i64)row.x * a.table_stride + e.c];
      }
      e.next(sh.step());
    }
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      const bool keeps = (at[j] & 6) == 6;  // its own whole page: not held any less
      if (keeps) now[j] = before[j];
      if (at[j] & 1 && !keeps) {
        if (ae_in_pool(before[j], a.num_pages))
          ae_set_bit(st.held, before[j]);
        else
          bad |= 16u;
      }
      if (at[j] & 2) {
        if (ae_in_pool(now[j], a.num_pages))
          ae_set_bit(st.whole, now[j]);
        else
          bad |= 16u;
      }
      if (at[j] & 8) a.table_out[i0 + j * sh.step()] = now[j];
    }
  }
  if (bad) atomicOr(a.status, bad);
}

AE_DEVICE void ae_fork_lists(const AePlanForksArgs& a, const AeListState& st, const AeListShare sh) {
  const int tid = (int)threadIdx.x, P = 1 << a.page_log2, B = a.B, W = a.max_pages;
  const int head = min(max(*a.free_head, 0), a.n_free);
  // rows that copy in front of a thread's share, 8 rows at most
  const int per = (B + AE_LIST_THREADS - 1) / AE_LIST_THREADS, r0 = min(tid * per, B), r1 = min(r0 + per, B);
  u32 copy = 0;  // of row r0 + j: bit j
  for (int r = r0; r < r1; ++r) {
    const int4 row = st.rows[r];
    if (row.z >= 0 && ((ae_word(st.whole + (row.z >> 5)) >> (row.z & 31) & 1) || ae_word(st.owner + row.z) != AE_FORK_KEY(r, row.x))) copy |= 1u << (r - r0);
  }
  int taken, before, all_freed;
  int order = ae_cta_scan(__popc(copy), taken);
  // pages that are held no more
  auto freed = [&](int w) { return ae_word(st.held + w) & ~(ae_word(st.whole + w) | ae_word(st.begun + w)); };
  const int share = (a.words + sh.ctas - 1) / sh.ctas, w0 = min(sh.cta * share, a.words), w1 = min(w0 + share, a.words);
  ae_count_bits(a.words, w0, freed, before, all_freed);
  // got: taken from the list; reused: of the freed ones, the first; page reused + j of those stands at top + j, as far as there is room
  const int got = min(taken, a.n_free - head), reused = min(taken - got, all_freed), back = all_freed - reused;
  const int top = max(head + got - back, 0), room = head + got - top;
  if (reused > 0)  // the rows that copy into freed pages; read behind a barrier of ae_each_page
    for (int r = r0, i = order - got; r < r1; ++r)
      if (copy >> (r - r0) & 1) {
        if (i >= 0 && i < reused) st.reusing[i] = (u16)r;
        ++i;
      }
  ae_each_page(w0, w1, before, freed, [&](int page, bool is, int j) {
    if (!is) return;
    if (j >= reused) {
      if (j - reused < room) a.free_out[top + j - reused] = page;
      return;
    }
    const int r = st.reusing[j];
    const int4 row = st.rows[r];
    const AePageCopy e = {row.z, page, row.y & (P - 1), 0};
    a.copies[got + j] = e;
    a.table_out[(i64)r * W + (row.y >> a.page_log2)] = page;
  });
  for (u32 i = sh.first(); i < (u32)a.n_free; i += sh.step())
    if ((int)i < top || (int)i >= top + room) a.free_out[i] = a.free_pages[i];
  u32 bad = back > room ? 4u : 0u;
  for (int r = r0; r < r1; ++r) {
    const bool copies = copy >> (r - r0) & 1;
    const int mine = order;
    order += copies;
    if (r % sh.ctas != sh.cta) continue;
    const int4 row = st.rows[r];
    int n = row.y;
    const int part = n & (P - 1);
    if (row.z >= 0 && !(copies && mine >= got && mine < got + reused)) {
      int page = row.z;
      if (copies) {
        const bool there = mine < got;
        page = there ? a.free_pages[head + mine] : -1;
        AePageCopy e = {row.z, page, part, 0};
        if (!ae_in_pool(page, a.num_pages)) {  // no page: the row ends with its whole ones
          bad |= there ? 16u : 1u;
          n -= part;
          page = 0;
          // the list ends where the free pages did; a page outside the pool leaves no gap in it
          e.dst = e.src;
          if (!there) e.src = e.dst = e.slots = 0;
        }
        a.copies[mine] = e;
      }
      a.table_out[(i64)r * W + (row.y >> a.page_log2)] = page;
    }
    a.lens_out[r] = n;
  }
  for (u32 i = sh.first() + taken; i < (u32)B; i += sh.step()) {
    const AePageCopy none = {0, 0, 0, 0};
    a.copies[i] = none;
  }
  if (bad) atomicOr(a.status, bad);
  if (sh.first() == 0) *a.head_out = top;
}

extern "C" __global__ void __launch_bounds__(AE_LIST_THREADS) ae_plan_forks(const __grid_constant__ AePlanForksArgs a) {
  const AeListShare sh = {(int)blockIdx.x, (int)gridDim.x};
  AeListState st;
#if AE_PHASE == 0 || AE_PHASE == 3
  __shared__ u16 reusing[4096];
  st.reusing = reusing;
#endif
#if AE_PHASE == 0
  extern __shared__ uint4 smem_raw[];
  st.rows = (int4*)smem_raw;
  st.held = (u32*)(st.rows + a.B);
#else
  st.rows = a.rows;
  st.held = a.held;
#endif
  st.whole = st.held + a.words;
  st.begun = st.whole + a.words;
  st.owner = st.begun + a.words;
  st.holes = nullptr;
  ae_grid_wait();  // brought up under the kernel in front
  ae_grid_trigger();
#if AE_PHASE == 0
  ae_fork_rows(a, st, sh);
  __syncthreads();
  ae_fork_marks(a, st, sh);
  __syncthreads();
  ae_fork_lists(a, st, sh);
#elif AE_PHASE == 1
  ae_fork_rows(a, st, sh);
#elif AE_PHASE == 2
  ae_fork_marks(a, st, sh);
#else
  ae_fork_lists(a, st, sh);
#endif
}
