// Moves every page in use to the front of its pool: with U pages in use, those from U on go into the unused ones below it, both in ascending order.
// Written are the block tables with the new numbers, the list of copies {page, new page, slots in use} and the free list (all pages, U of them taken).
//
// One word a page holds how many of its slots the rows use (a maximum, so the order of the atomics does not show), then for a page that moves its place in
// the list.  One running sum over the pages serves both sides: x is hole number x - (in use below x), or mover number (in use below x) - (in use
// below U).  Holes write the list's second number, moving pages the others.
// Expects AE_LIST_THREADS, AE_LIST_CTAS, AE_LIST_BATCH (table entries of a thread on their way together).
extern "C" __global__ void __launch_bounds__(AE_LIST_THREADS) ae_plan_compaction(const __grid_constant__ AePlanCompactionArgs a) {
  __shared__ int warp_sum[2][AE_LIST_THREADS / 32];
  __shared__ u32 sm_bad;
  ae_grid_wait();
  ae_grid_trigger();
  const int cta = (int)cluster_ctarank(), tid = (int)threadIdx.x, lane = tid & 31;
  const int gtid = cta * AE_LIST_THREADS + tid, gstep = AE_LIST_CTAS * AE_LIST_THREADS;
  const int P = 1 << a.page_log2, B = a.B, W = a.max_pages, groups = (a.num_pages + 3) / 4;
  const i64 most = (i64)W << a.page_log2;
  u32 bad = 0;
  if (tid == 0) sm_bad = 0;
  if (gtid == 0) *a.status = 0;
  for (int i = gtid; i < groups; i += gstep) ((uint4*)a.state)[i] = make_uint4(0, 0, 0, 0);
  for (int i = gtid; i < a.n_copies; i += gstep) ((uint4*)a.copies)[i] = make_uint4(0, 0, 0, 0);
  for (int i = gtid; i < a.num_pages; i += gstep) a.free_out[i] = i;
  ae_phase_end();

  // how many slots of each page are in use
  const int warps = gstep / 32, chunks = (W + 31) / 32, gwarp = cta * (AE_LIST_THREADS / 32) + (tid >> 5);
  auto tokens_of = [&](int len) { return min((i64)max(len, 0), most); };
  for (int i0 = gwarp; i0 < B * chunks; i0 += warps * AE_LIST_BATCH) {
    int page[AE_LIST_BATCH], slots[AE_LIST_BATCH];
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {  // the reads in front of the atomics, which the compiler moves no read across
      page[j] = slots[j] = 0;
      const int i = i0 + j * warps;
      if (i >= B * chunks) continue;
      const int r = i / chunks, c = (i - r * chunks) * 32 + lane, len = a.lens[r];
      if (c == 0) bad |= len < 0 ? 8u : len > most ? 2u : 0u;
      slots[j] = c < W ? (int)min(max(tokens_of(len) - ((i64)c << a.page_log2), (i64)0), (i64)P) : 0;
      if (slots[j]) page[j] = a.table[(i64)r * a.table_stride + c];
    }
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      if (!slots[j]) continue;
      if (page[j] >= 0 && page[j] < a.num_pages)
        atomicMax(a.state + page[j], (u32)slots[j]);
      else
        bad |= 16u;
    }
  }
  ae_phase_end();

  // pages in use in front of a thread's share
  int first, end, mine = 0;
  ae_page_share(a.num_pages, cta, first, end);
  const int share = (end - first) / 4, tper = (share + AE_LIST_THREADS - 1) / AE_LIST_THREADS;
  const int g0 = first / 4 + min(tid * tper, share), g1 = min(g0 + tper, end / 4);
#pragma unroll 4
  for (int g = g0; g < g1; ++g) {
    const uint4 u = __ldcg((const uint4*)a.state + g);
    mine += (u.x != 0) + (u.y != 0) + (u.z != 0) + (u.w != 0);
  }
  int cta_used, used = 0;
  int before = ae_cta_scan(mine, warp_sum[0], cta_used);
  if (tid == 0) a.counts[cta] = cta_used;
  if (bad) atomicOr(&sm_bad, bad);
  ae_phase_end();
#pragma unroll
  for (int i = 0; i < AE_LIST_CTAS; ++i) {
    const int n = __ldcg(a.counts + i);
    if (i < cta) before += n;
    used += n;
  }
  // those below page `used`: whole shares, and a part of the one that it lies in, counted by every CTA for itself
  int below = 0, part = 0;
  for (int i = 0; i < AE_LIST_CTAS; ++i) {
    int f, e;
    ae_page_share(a.num_pages, i, f, e);
    if (e <= used)
      below += __ldcg(a.counts + i);
    else if (f < used)
      for (int x = f + tid; x < used; x += AE_LIST_THREADS) part += __ldcg(a.state + x) != 0;
  }
  ae_cta_scan(part, warp_sum[1], part);
  below += part;
  for (int g = g0; g < g1; ++g) {
    const uint4 u = __ldcg((const uint4*)a.state + g);
    const u32 w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int page = g * 4 + k;
      if (page >= a.num_pages) break;
      if (w[k]) {
        const int place = before++ - below;
        if (page >= used) {
          a.copies[place].src = page;
          a.copies[place].slots = (int)w[k];
          a.state[page] = (u32)place;
        }
      } else if (page < used) {
        a.copies[page - before].dst = page;
      }
    }
  }
  if (gtid == 0) *a.head_out = used;
  if (tid == 0 && sm_bad) atomicOr(a.status, sm_bad);
  ae_phase_end();

  // the tables with the new numbers
  for (int i0 = gwarp; i0 < B * chunks; i0 += warps * AE_LIST_BATCH) {
    int page[AE_LIST_BATCH], place[AE_LIST_BATCH];
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      page[j] = 0;
      const int i = i0 + j * warps;
      if (i >= B * chunks) continue;
      const int r = i / chunks, c = (i - r * chunks) * 32 + lane;
      if (c < W && ((i64)c << a.page_log2) < tokens_of(a.lens[r])) page[j] = a.table[(i64)r * a.table_stride + c];
    }
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) place[j] = page[j] >= used && page[j] < a.num_pages ? (int)__ldcg(a.state + page[j]) : -1;
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j)
      if (place[j] >= 0) page[j] = __ldcg(&a.copies[place[j]].dst);
#pragma unroll
    for (int j = 0; j < AE_LIST_BATCH; ++j) {
      const int i = i0 + j * warps;
      if (i >= B * chunks) break;
      const int r = i / chunks, c = (i - r * chunks) * 32 + lane;
      if (c < W) a.table_out[(i64)r * W + c] = page[j];
    }
  }
}
