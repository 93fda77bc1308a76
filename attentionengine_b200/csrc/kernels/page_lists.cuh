// What the planners of a pool's pages share.  A plan is a few phases over the rows' table entries and over bitmaps of the pages, each of which needs all
// of the one in front of it.  AE_PHASE 0: one CTA runs them all, with what passes between them in its shared memory, for small tables (latency: an L2
// round trip and a launch less for each phase); n > 0: a launch for each over the whole GPU, brought up under the one in front, with it in a workspace.
//
// Bitmaps because the numbering of freed or moved pages is a running sum over the pool: 32 pages a word, so every CTA makes the sums in front of its
// share of the words for itself.  Bits are set by atomics whose order does not show.
// Expects AE_LIST_THREADS, AE_LIST_BATCH (table entries of a thread on their way together), AE_PHASE.

struct AeListShare {
  int cta, ctas;
  AE_DEVICE u32 first() const { return cta * AE_LIST_THREADS + threadIdx.x; }
  AE_DEVICE u32 step() const { return ctas * AE_LIST_THREADS; }
};

// What passes between the phases: in shared memory behind each other, or the launch's workspace.
struct AeListState {
  int4* rows;                 // [B] of the forks
  u32 *held, *whole, *begun;  // [words] each, behind each other
  u32* owner;                 // [num_pages] of begun pages: a key, or slots; of moving pages: their place in the list
  int* holes;                 // [num_pages / 2] pages that moving ones take, by place; null: the list's
  u16* reusing;               // [B] of the forks, in shared memory: rows that copy into pages which the step gives back
};
AE_DEVICE u32 ae_word(const u32* p) {  // written by another phase
#if AE_PHASE == 0
  return *p;
#else
  return __ldcg(p);
#endif
}
AE_DEVICE void ae_set_bit(u32* bits, int page) { atomicOr(bits + (page >> 5), 1u << (page & 31)); }
AE_DEVICE bool ae_in_pool(int page, int num_pages) { return page >= 0 && page < num_pages; }

// A thread's entries of a [B, W] table, AE_LIST_BATCH at a time: (r, c) without a division for each.
struct AeEntries {
  u32 i, total, W, dr, dc;
  int r, c;
  AE_DEVICE AeEntries(const AeListShare& s, int B, int W_) : i(s.first()), total((u32)B * (u32)W_), W(W_), dr(s.step() / W_), dc(s.step() % W_) {
    r = (int)(i / W);
    c = (int)(i % W);
  }
  AE_DEVICE bool more() const { return i < total; }
  AE_DEVICE void next(u32 step) {
    i += step;
    r += dr;
    c += dc;
    if (c >= (int)W) c -= W, ++r;
  }
};

// Exclusive sum over the CTA's threads; `total` is the whole.
AE_DEVICE int ae_cta_scan(int x, int& total) {
  __shared__ int warp_sum[AE_LIST_THREADS / 32];
  const u32 lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, s, o);
    if ((int)lane >= o) s += y;
  }
  __syncthreads();  // the sums of the scan in front have been read
  if (lane == 31) warp_sum[warp] = s;
  __syncthreads();
  const int w = lane < AE_LIST_THREADS / 32 ? warp_sum[lane] : 0;
  total = __reduce_add_sync(0xffffffffu, w);
  return __reduce_add_sync(0xffffffffu, lane < warp ? w : 0) + s - x;
}

// Sums of the bits of `word(w)` over all words: in front of word `at`, and all.
template <class F>
AE_DEVICE void ae_count_bits(int words, int at, F&& word, int& before, int& all) {
  int b = 0, n = 0;
#pragma unroll 4
  for (int w = threadIdx.x; w < words; w += AE_LIST_THREADS) {
    const int k = __popc(word(w));
    n += k;
    if (w < at) b += k;
  }
  ae_cta_scan(b, before);
  ae_cta_scan(n, all);
}

// emit(page, whether its bit is set, set bits in front of it) for each page of words [from, to), with `before` set bits in front of those; a warp takes a
// word, a lane a page.
template <class F, class G>
AE_DEVICE void ae_each_page(int from, int to, int before, F&& word, G&& emit) {
  __shared__ u32 bits[AE_LIST_THREADS];
  __shared__ int base[AE_LIST_THREADS];
  const int tid = threadIdx.x, lane = tid & 31;
  for (int w0 = from; w0 < to; w0 += AE_LIST_THREADS) {
    const u32 mine = w0 + tid < to ? word(w0 + tid) : 0u;
    int n;
    const int at = before + ae_cta_scan(__popc(mine), n);  // its barriers: the words in front have been read
    bits[tid] = mine;
    base[tid] = at;
    __syncthreads();
    for (int i = tid >> 5; i < min(to - w0, AE_LIST_THREADS); i += AE_LIST_THREADS / 32) {
      const u32 b = bits[i];
      emit((w0 + i) * 32 + lane, (b >> lane & 1) != 0, base[i] + __popc(b & ((1u << lane) - 1)));
    }
    before += n;
    __syncthreads();
  }
}
