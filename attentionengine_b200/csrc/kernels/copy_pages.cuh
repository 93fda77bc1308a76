// Copies the first slots of pages into other pages, in every pool of a launch: keys, values and scales of all layers at once.
//
// A copy's bytes are cut into parts, and a CTA takes parts in turn: one load of the list's entry, then sixteen loads a thread in front of their
// stores.  HBM-bound once a few hundred parts are under way: 1500 pages of 64 tokens, 8 heads of 128 dims, in four layers (1.5 GB
// in and out) 251 us, 6.1 TB/s; 96 begun ones in eight layers (96 MB) 18.4 us, 5.2 TB/s.  Eight reads a thread in 256 of them, 257 and 20.8; four, 283 and 25; parts of
// 8 KB, 275 and 25.5, of 64 KB, 248 and 20.2.  Which page goes where and how many slots stands on the device; a list ends at
// its first entry without slots, which every CTA looks for itself, 256 entries a step, before it copies anything: 2 to 5 ns an entry.  That is next to nothing for a
// list of 1500 pages of 64 KB, and the larger part for long lists of small pages: in a graph, 1500 entries of 1 KB 5.9 us, 16300 of them 86 us, 16300 of 16 KB (534 MB) 162 us, in
// eight pools (4.3 GB) 757 us, 5.6 TB/s.  Entries that name a page outside the pool, or more slots than a page has, are passed over.
// An access is as wide as a slot's bytes and place allow (16, 4, 2 or 1), in slots that lie behind each other too, so odd slots take up to 16 times the
// instructions.
// A build for pools whose slots lie behind each other (AE_COPY_RUNS), and one for others, whose places take registers of their own: 1200 pages whose 8 heads lie
// one behind the other 27.5 to 28.5 us, 5.5 TB/s (37 with both in one build, 85 without reads in front of the writes).  Seven CTAs an SM at least: left to the compiler 173
// registers, the begun pages 21.4 us.
// Expects AE_COPY_THREADS, AE_COPY_UNROLL (reads of a thread in front of its writes), AE_COPY_RUNS.

// n units of V, from the unit `from` on of a page's part.  A pool's slots are runs of `per` units, row_st bytes apart, `rows` of them in slot_st bytes.
template <typename V>
AE_DEVICE void ae_copy_part(const AeCopyPool& p, const u8* src, u8* dst, int from, int n) {
#if AE_COPY_RUNS
  src += (i64)from * sizeof(V);
  dst += (i64)from * sizeof(V);
  for (int i = threadIdx.x; i < n; i += AE_COPY_THREADS * AE_COPY_UNROLL) {
    V v[AE_COPY_UNROLL];
#pragma unroll
    for (int u = 0; u < AE_COPY_UNROLL; ++u)
      if (i + u * AE_COPY_THREADS < n) v[u] = __ldcs((const V*)src + i + u * AE_COPY_THREADS);
#pragma unroll
    for (int u = 0; u < AE_COPY_UNROLL; ++u)
      if (i + u * AE_COPY_THREADS < n) __stcs((V*)dst + i + u * AE_COPY_THREADS, v[u]);
  }
#else
  const int per = p.run / (int)sizeof(V), end = from + n;
  for (int i0 = from + threadIdx.x; i0 < end; i0 += AE_COPY_THREADS * AE_COPY_UNROLL) {
    V v[AE_COPY_UNROLL];
    i64 at[AE_COPY_UNROLL];
#pragma unroll
    for (int u = 0; u < AE_COPY_UNROLL; ++u) {
      const int i = min(i0 + u * AE_COPY_THREADS, end - 1), row = i / per, slot = row / p.rows;
      at[u] = slot * p.slot_st + (row - slot * p.rows) * p.row_st + (i64)(i - row * per) * sizeof(V);
      v[u] = __ldcs((const V*)(src + at[u]));
    }
#pragma unroll
    for (int u = 0; u < AE_COPY_UNROLL; ++u)
      if (i0 + u * AE_COPY_THREADS < end) __stcs((V*)(dst + at[u]), v[u]);
  }
#endif
}

// Entries in front of the first without slots.
AE_DEVICE int ae_list_length(const AePageCopy* copies, int most) {
  __shared__ int red[AE_COPY_THREADS / 32];
  for (int base = 0; base < most; base += 4 * AE_COPY_THREADS) {
    int end = most;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const int i = base + j * AE_COPY_THREADS + (int)threadIdx.x;
      if (i < most && copies[i].slots <= 0) end = i;
    }
    end = __reduce_min_sync(0xffffffffu, end);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = end;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < AE_COPY_THREADS / 32; ++w) end = min(end, red[w]);
    if (end < most) return end;
    __syncthreads();  // `red` has been read
  }
  return most;
}

extern "C" __global__ void __launch_bounds__(AE_COPY_THREADS, 7) ae_copy_pages(const __grid_constant__ AeCopyPagesArgs a) {
  ae_grid_wait();
  ae_grid_trigger();
  const i64 items = (i64)ae_list_length(a.copies, a.n_copies) * a.parts;
  for (i64 item = blockIdx.x; item < items; item += gridDim.x) {
    const int c = (int)(item / a.parts), part = (int)(item - (i64)c * a.parts);
    const AePageCopy e = a.copies[c];
    if (e.src < 0 || e.src >= a.num_pages || e.dst < 0 || e.dst >= a.num_pages || e.slots > a.page_size) continue;
    int i = 0;
    while (i + 1 < a.n_pools && part >= a.pools[i + 1].first) ++i;
    const AeCopyPool& p = a.pools[i];
    const int s0 = (part - p.first) * p.slots_part, s1 = min(s0 + p.slots_part, e.slots);
    if (s0 == 0 && p.extra)
      for (int k = threadIdx.x * 4; k < p.extra_bytes; k += AE_COPY_THREADS * 4)
        *(u32*)(p.extra + (i64)e.dst * p.extra_st + k) = *(const u32*)(p.extra + (i64)e.src * p.extra_st + k);
    if (s0 >= s1) continue;
    const u8* const src = p.base + (i64)e.src * p.page_st;
    u8* const dst = p.base + (i64)e.dst * p.page_st;
    const int slot = p.rows * (p.run / p.vec);  // units of a slot
    if (p.vec == 16)
      ae_copy_part<uint4>(p, src, dst, s0 * slot, (s1 - s0) * slot);
    else if (p.vec == 4)
      ae_copy_part<u32>(p, src, dst, s0 * slot, (s1 - s0) * slot);
    else if (p.vec == 2)
      ae_copy_part<u16>(p, src, dst, s0 * slot, (s1 - s0) * slot);
    else
      ae_copy_part<u8>(p, src, dst, s0 * slot, (s1 - s0) * slot);
  }
}
