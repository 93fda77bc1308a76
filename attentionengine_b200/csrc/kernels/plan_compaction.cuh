// Moves every page in use to the front of its pool: with U pages in use, those from U on go into the unused ones below it, both in ascending order.
// Written are the block tables with the new numbers, the list of copies {page, new page, slots in use} and the free list (all pages, U of them taken).
//
// Phase 1 clears the bitmaps and the slots of begun pages; phase 2 sets the pages' bits (held whole, begun) and takes the maximum of a begun page's slots; in
// phase 3 one running sum over the pages serves both sides: page x is hole number x - (in use below x), or mover number (in use below x) - (in use below
// U), and holes write the list's second number, moving pages the others; phase 4 writes the tables, from the places that phase 3 wrote.

AE_DEVICE int ae_len(const AePlanCompactionArgs& a, int r) {  // in the table
  return (int)min((i64)max(a.lens[r], 0), (i64)a.max_pages << a.page_log2);
}

AE_DEVICE void ae_pack_rows(const AePlanCompactionArgs& a, const AeListState& st, const AeListShare sh) {
  if (sh.first() == 0) *a.status = 0;
  for (u32 i = sh.first(); i < 2u * (u32)a.words / 4; i += sh.step()) ((uint4*)st.whole)[i] = make_uint4(0, 0, 0, 0);
  for (u32 r = sh.first(); r < (u32)a.B; r += sh.step()) {
    const int n = ae_len(a, (int)r);
    if (n & ((1 << a.page_log2) - 1)) {
      const int page = a.table[(i64)r * a.table_stride + (n >> a.page_log2)];
      if (ae_in_pool(page, a.num_pages)) st.owner[page] = 0;
    }
  }
  for (u32 i = sh.first(); i < (u32)a.n_copies; i += sh.step()) ((uint4*)a.copies)[i] = make_uint4(0, 0, 0, 0);
  for (u32 i = sh.first(); i < (u32)a.num_pages; i += sh.step()) a.free_out[i] = (int)i;
}

AE_DEVICE void ae_pack_marks(const AePlanCompactionArgs& a, const AeListState& st, const AeListShare sh) {
  const int P = 1 << a.page_log2;
  u32 bad = 0;
  for (AeEntries e(sh, a.B, a.max_pages); e.more();) {
    int page[AE_LIST_BATCH], slots[AE_LIST_BATCH];
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {  // the reads in front of the atomics, which the compiler moves no read across
      page[j] = slots[j] = 0;
      if (e.more()) {
        const int n = ae_len(a, e.r);
        if (e.c == 0) bad |= a.lens[e.r] < 0 ? 8u : a.lens[e.r] > n ? 2u : 0u;
        if (e.c < (int)(((i64)n + P - 1) >> a.page_log2)) {
          slots[j] = min(n - (e.c << a.page_log2), P);
          page[j] = a.table[(i64)e.r * a.table_stride + e.c];
        }
      }
      e.next(sh.step());
    }
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      if (!slots[j]) continue;
      if (!ae_in_pool(page[j], a.num_pages)) {
        bad |= 16u;
      } else if (slots[j] == P) {
        ae_set_bit(st.whole, page[j]);
      } else {
        ae_set_bit(st.begun, page[j]);
        atomicMax(st.owner + page[j], (u32)slots[j]);
      }
    }
  }
  if (bad) atomicOr(a.status, bad);
}

AE_DEVICE int ae_pack_lists(const AePlanCompactionArgs& a, const AeListState& st, const AeListShare sh) {
  auto in_use = [&](int w) { return ae_word(st.whole + w) | ae_word(st.begun + w); };
  const int share = (a.words + sh.ctas - 1) / sh.ctas, w0 = min(sh.cta * share, a.words), w1 = min(w0 + share, a.words);
  int before, used, below, all;
  ae_count_bits(a.words, w0, in_use, before, used);
  auto low = [&](int w) { return w * 32 + 32 <= used ? 0xffffffffu : w * 32 >= used ? 0u : (1u << (used & 31)) - 1; };  // pages below `used`
  ae_count_bits(a.words, a.words, [&](int w) { return in_use(w) & low(w); }, below, all);
  ae_each_page(w0, w1, before, in_use, [&](int page, bool is, int j) {
    if (page < used && !is) {
      a.copies[page - j].dst = page;
      if (st.holes) st.holes[page - j] = page;
    } else if (page >= used && is) {
      const int place = j - below;
      const bool whole = ae_word(st.whole + (page >> 5)) >> (page & 31) & 1;
      a.copies[place].src = page;
      a.copies[place].slots = whole ? 1 << a.page_log2 : (int)ae_word(st.owner + page);
      st.owner[page] = (u32)place;
    }
  });
  if (sh.first() == 0) *a.head_out = used;
  return used;
}

AE_DEVICE void ae_pack_tables(const AePlanCompactionArgs& a, const AeListState& st, const AeListShare sh, int used) {
  for (AeEntries e(sh, a.B, a.max_pages); e.more();) {
    int page[AE_LIST_BATCH], place[AE_LIST_BATCH];
    bool moves[AE_LIST_BATCH];  // only pages of a row have a place: with none in use, the 0 of an entry behind its row is not below `used` either
    const u32 i0 = e.i;
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      moves[j] = e.more() && (i64)e.c << a.page_log2 < ae_len(a, e.r);
      page[j] = moves[j] ? a.table[(i64)e.r * a.table_stride + e.c] : 0;
      e.next(sh.step());
    }
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) place[j] = moves[j] && page[j] >= used && page[j] < a.num_pages ? (int)ae_word(st.owner + page[j]) : -1;
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j)
      if (place[j] >= 0) page[j] = st.holes ? st.holes[place[j]] : __ldcg(&a.copies[place[j]].dst);
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j)
      if (i0 + j * sh.step() < e.total) a.table_out[i0 + j * sh.step()] = page[j];
  }
}

extern "C" __global__ void __launch_bounds__(AE_LIST_THREADS) ae_plan_compaction(const __grid_constant__ AePlanCompactionArgs a) {
  const AeListShare sh = {(int)blockIdx.x, (int)gridDim.x};
  AeListState st;
  st.rows = nullptr;
#if AE_PHASE == 0
  extern __shared__ uint4 smem_raw[];
  st.held = (u32*)smem_raw;
#else
  st.held = a.held;
#endif
  st.whole = st.held;
  st.begun = st.whole + a.words;
  st.owner = st.begun + a.words;
  st.holes = AE_PHASE == 0 ? (int*)(st.owner + a.num_pages) : nullptr;
  ae_grid_wait();  // brought up under the kernel in front
  ae_grid_trigger();
#if AE_PHASE == 0
  ae_pack_rows(a, st, sh);
  __syncthreads();
  ae_pack_marks(a, st, sh);
  __syncthreads();
  const int used = ae_pack_lists(a, st, sh);
  __syncthreads();
  ae_pack_tables(a, st, sh, used);
#elif AE_PHASE == 1
  ae_pack_rows(a, st, sh);
#elif AE_PHASE == 2
  ae_pack_marks(a, st, sh);
#elif AE_PHASE == 3
  ae_pack_lists(a, st, sh);
#else
  ae_pack_tables(a, st, sh, __ldcg(a.head_out));
#endif
}
