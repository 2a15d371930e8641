// Attention of single tokens over a cache in eight bits (kv8.cuh) on the tensor cores: bfloat16 queries, head size 64 or 128, up to 16
// query heads a kv head.
//
// A single token reads every code once, so the kernel has to keep HBM busy: 16.1 KB a page and kv head at head size 128 against
// 0.5 M operations.  Everything is done by warps on their own:
//   * The visible pages of all (sequence, kv head) pairs are one line of items; each block takes an equal stretch of it, and each of its
//     warps an equal stretch of that, whatever the sequences' lengths are.  A pair that several warps share is joined by those warps at the
//     block's end, one that several blocks share by a second, small kernel.  Where every pair has a block and no more than two pages a warp,
//     blocks take pairs instead and there is no second kernel.
//   * A warp has its own ring of shared memory, filled by untiled bulk copies (K and V tile of a page are one stretch of memory each;
//     no tensor map; the exponents come by cp.async three items ahead, since a bulk copy of 64 bytes costs as much to ask for as one of 8 KB), and no barrier with other warps on the way.  K and V take turns in the slots, so a slot is free again after half a page.
//   * q k^T: m16n8k32 on the codes as they are.  A bfloat16 query (8 bits of mantissa) is the sum of TWO e4m3 numbers of 4 bits each: the
//     G <= 8 heads' larger parts are the fragment's rows 0-7, the rests rows 8-15 that would be idle, and the two results are added.  Queries
//     are scaled by a power of two so that the row's largest lies in 2^7 .. 2^8: elements down to 2^-9 of that are exact, smaller ones off by at
//     most 2^-18 of it.  (m16n8k32 of e4m3 issues at 0.97 an SM and clock, m16n8k16 of f16 at 0.5, a pair of conversions to f16 at 0.67.)
//     The order of the inner axis is free as long as both operands agree, so a thread takes 16 neighbouring codes of a key in one 16-byte
//     load and the query's elements to match.
//   * p v: m16n8k16 in half precision (e4m3 becomes that exactly), 16 dims of V as M and 8 heads as N, so that no row is idle.  Values lie dim by
//     dim, and with keys dealt to the scores' columns as 16 t + 2 j + i the scores a thread holds are exactly the weights its fragments need,
//     and the exponents of its 16 keys are one 16-byte load.  Nothing moves between lanes but the rows' maxima.
//   * A value's power of two joins the weight before it is rounded: with x the score (base 2) and E the exponent, weights are 2^(x - m) in
//     the denominator, and 2^(x + E - M + 15) in half precision beside the codes, with M the running maximum of x + E.  So a large value
//     of next to no weight takes nothing from the precision of the others; weights from 1 down to 2^-29 of the row's largest x + E keep all 11 bits.
//
// Measured (replayed graphs, other inputs each time; 32 heads over 8 of 128 unless said): one sequence of 131,072 keys 52.5 us, 5.2 TB/s; 8 x 4,096 keys 16.3;
// one of 301 keys 7.9; 64 sequences seeing 1,000 keys, 64 heads over 8 of 64, 26.0.  With parts left out in a copy (of a state that took 53.1, 18.4, 7.8 and 29.7), us of these
// four: copies alone 41.8, 10.5, 3.9, 15.3; without the products and the softmax 45.9, 15.6, 5.1, 24.3.  So a long line of pages is bound by HBM, a short one by its start (lengths, places, the first
// pages: 3 us, cold code), the joins (1 to 1.5 us in the block, 1.5 to 3 of the second kernel) and what a warp does once a pair (its query's two parts, its end).
//
// Every wait on an mbarrier is bounded; one that runs out sets the library's status word (sx_kv8_decode_status).
#include "kv8.cuh"

#define KD_MAX_SEQS 2048
#define KD_FEW_SEQS 128          // every warp looks at all lengths by itself
#define KD_SPIN_LIMIT (1u << 26)
#define KD_DOWN 3.0517578125e-5f      // 2^-15
#define KD_DESC 64               // items a warp knows ahead: two batches of 32
#define KD_LOG2E 1.44269504f

// Three warps a scheduler hide one another's latencies: a page takes a warp alone 3,400 clocks, and HBM delivers one to an SM every 710 (four at head
// size 64 and three slots each: 33.0 us for 64 sequences seeing 1,000 keys where three took 31.5, 26.0 by now).  With more than 8 heads a kv head a thread has two
// rows' registers, and there are two.
template <int HD, bool MORE> struct KdLayout {
  static constexpr int WARPS = MORE ? 8 : 12;
  static constexpr int TILE = SX_PAGE * HD;
  static constexpr int SLOTS = (MORE ? 3 : 2) * (128 / HD);
  static constexpr int AHEAD = 3;                               // items whose exponents (and at most whose tiles) are under way ahead of the one at work
  static constexpr int EXPS = 2 * SX_PAGE;                      // an item's exponents of keys and values
  static constexpr int PART = HD + 2;                           // a row's maximum, sum and result
  static constexpr int RING = WARPS * SLOTS * TILE;
  static constexpr int FIXED = RING + WARPS * (KD_DESC * (int)sizeof(int4) + (AHEAD + 1) * EXPS);       // ... and the starts of the sequences' items behind it
};
#define KD_MAX_WARPS 12

struct KdArgs {
  const bf16* q;
  bf16* out;
  const uint8_t *k, *v, *ke, *ve;
  const int *seq_lens, *row_seq, *block_table;                  // of row s: keys it may see less len_add, its row of the table (null: s)
  const float* sinks;
  float* part;                 // results of pairs' parts [warps, then 2 a block][rows of a kv head][HD + 2]: maximum, sum, the row
  int* status;
  int len_add, maxp, n_pages, S, nh, nkv, window, blocks, warps, by_pair;
  float scale;
};

__device__ __forceinline__ uint32_t kd_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool kd_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t i = 0; i < KD_SPIN_LIMIT; ++i) {
    uint32_t ok;
    asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
  }
  return false;
}
__device__ __forceinline__ void kd_copy(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
// first visible page of a sequence of that length and one behind its last
__device__ __forceinline__ int2 kd_range(const KdArgs& a, int len) {
  const int first = a.window > 0 ? max(0, len - a.window) >> 6 : 0;
  return make_int2(first, max(first, min((len + 63) >> 6, a.maxp)));
}
// start[s]: pages of the sequences before s, start[S] of all, for one kv head; every thread of the block takes part
template <int THREADS>
__device__ __forceinline__ void kd_starts(const KdArgs& a, int* start, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int before = 0;
  for (int s0 = 0; s0 < a.S; s0 += THREADS) {
    const int s = s0 + threadIdx.x;
    int n = 0;
    if (s < a.S) {
      const int2 r = kd_range(a, a.seq_lens[s] + a.len_add);
      n = r.y - r.x;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int total = 0, mine = before;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w < warp) mine += warp_sums[w];
      total += warp_sums[w];
    }
    if (s < a.S) start[s] = mine + x - n;
    before += total;
    __syncthreads();
  }
  if (threadIdx.x == 0) start[a.S] = before;
  __syncthreads();
}
// the same by a warp for itself
__device__ __forceinline__ void kd_starts_warp(const KdArgs& a, int* start) {
  const int lane = threadIdx.x & 31;
  int len[KD_FEW_SEQS / 32], before = 0;
#pragma unroll
  for (int i = 0; i < KD_FEW_SEQS / 32; ++i) len[i] = 32 * i + lane < a.S ? a.seq_lens[32 * i + lane] : 0;
#pragma unroll
  for (int i = 0; i < KD_FEW_SEQS / 32; ++i) {
    const int s = 32 * i + lane;
    if (32 * i >= a.S) break;
    const int2 r = kd_range(a, len[i] + a.len_add);
    const int n = s < a.S ? r.y - r.x : 0;
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (s < a.S) start[s] = before + x - n;
    before += __shfl_sync(0xffffffffu, x, 31);
  }
  if (lane == 0) start[a.S] = before;
  __syncwarp();
}
// the blocks that work (a block of fewer items than warps would leave some idle), and the first item of block b
__device__ __forceinline__ int kd_workers(const KdArgs& a, int n) { return max(1, min(a.blocks, (n + a.warps - 1) / a.warps)); }
__device__ __forceinline__ int kd_first(int b, int n, int workers) {
  const int q = n / workers;
  return b * q + min(b, n - q * workers);
}
__device__ __forceinline__ int kd_worker_of(int item, int n, int workers) {
  const int q = n / workers, longer = (n - q * workers) * (q + 1);        // items of the blocks that have one more
  return item < longer ? item / (q + 1) : n - q * workers + (item - longer) / q;
}
// the sequence of item x: the last s with start[s] * nkv <= x among those that have pages
__device__ __forceinline__ int kd_seq_of(const int* start, int S, int nkv, int x) {
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] * nkv <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// MORE: more than 8 query heads a kv head (two rows of scores a thread, two tiles of heads in p v)
template <int HD, bool MORE>
__global__ void __launch_bounds__(KdLayout<HD, MORE>::WARPS * 32, 1) kv8_decode_kernel(const KdArgs a) {
  using L = KdLayout<HD, MORE>;
  constexpr int RP = MORE ? 2 : 1, WARPS = L::WARPS, FIRST = (L::SLOTS + 1) / 2;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[WARPS * L::SLOTS];
  __shared__ int warp_sums[WARPS], first_unit[WARPS], last_unit[WARPS], first_seq;
  int4* desc_all = reinterpret_cast<int4*>(smem + L::RING);
  unsigned char* exps = smem + L::RING + WARPS * KD_DESC * sizeof(int4) + (threadIdx.x >> 5) * (L::AHEAD + 1) * L::EXPS;
  int* start = reinterpret_cast<int*>(smem + L::RING + WARPS * (KD_DESC * sizeof(int4) + (L::AHEAD + 1) * L::EXPS));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < L::SLOTS; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(kd_smem(&bars[warp * L::SLOTS + s])));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  const bool few = a.S <= KD_FEW_SEQS;
  if (few) {
    start += warp * (a.S + 1);                                  // (a copy a warp)
    kd_starts_warp(a, start);
  } else {
    kd_starts<WARPS * 32>(a, start, warp_sums);
  }
  const int G = a.nh / a.nkv, n_all = start[a.S] * a.nkv;
  if (n_all == 0) {                                             // nobody sees anything
    for (size_t i = blockIdx.x * WARPS * 32 + threadIdx.x; i < (size_t)a.S * a.nh * HD; i += gridDim.x * WARPS * 32) a.out[i] = __float2bfloat16_rn(0.f);
    return;
  }
  // (Every instruction up to the first copy is latency: a kernel's code comes in cold, at some ten clocks an instruction.)
  int b0 = 0, b1 = 0;                                           // the block's items
  if (a.by_pair) {
    const int s = blockIdx.x / a.nkv, n = start[s + 1] - start[s];
    b0 = start[s] * a.nkv + (blockIdx.x - s * a.nkv) * n;
    b1 = b0 + n;
  } else {
    const int workers = max(1, min(a.blocks, (n_all + WARPS - 1) / WARPS));      // (as kd_workers)
    if (blockIdx.x < workers) {
      b0 = kd_first(blockIdx.x, n_all, workers);
      b1 = kd_first(blockIdx.x + 1, n_all, workers);
    }
  }
  auto first_of = [&](int w) { return b0 + (b1 - b0) * w / WARPS; };
  const int x0 = first_of(warp), n_items = first_of(warp + 1) - x0;
  int seq0 = 0;                                                 // a sequence at or before the first item's
  if (a.by_pair) {
    seq0 = blockIdx.x / a.nkv;
  } else if (few) {
#pragma unroll 1
    for (int s0 = 0; s0 < a.S; s0 += 32) seq0 += __popc(__ballot_sync(0xffffffffu, s0 + lane < a.S && start[s0 + lane + 1] * a.nkv <= x0));
  } else {
    for (int s = threadIdx.x; s < a.S; s += WARPS * 32)
      if (start[s] * a.nkv <= b0 && b0 < start[s + 1] * a.nkv) first_seq = s;
    __syncthreads();
    seq0 = first_seq;
  }
  int4* desc = desc_all + warp * KD_DESC;                       // (sequence, kv head, page of the sequence, page of the pool)
  unsigned char* ring = smem + warp * L::SLOTS * L::TILE;
  const uint32_t ring_a = kd_smem(ring), bar_a = kd_smem(&bars[warp * L::SLOTS]);
  // load number n of the warp: the K (even) or V (odd) tile of item n / 2, into slot n % SLOTS
  auto issue = [&](int n) {
    const int i = n >> 1;
    if (lane == 0 && i < n_items) {
      const int4 d = desc[i & (KD_DESC - 1)];
      const int slot = n % L::SLOTS;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar_a + slot * 8), "r"(L::TILE) : "memory");
      kd_copy(ring_a + slot * L::TILE, ((n & 1) ? a.v : a.k) + ((size_t)d.w * a.nkv + d.y) * L::TILE, L::TILE, bar_a + slot * 8);
    }
  };

  uint32_t qf[HD / 16][2][RP];                                  // [4 dims each][larger part, rest][row]
  float c[RP], m[RP], l[RP], M[RP], o[HD / 16][RP][4];          // o: dims 16 d + g (+ 8), heads 8 r + 2 t + {0, 1}
  int seq = -1, kvh = -1, unit_first = 0, unit0 = -1, len = 0;  // the pair at work, the item of the warp it began with; the warp's first pair
  auto begin = [&](int s, int h, int i) {
    seq = s; kvh = h; unit_first = i;
    len = a.seq_lens[s] + a.len_add;
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const int row = g + 8 * r;
      uint4 w[HD / 32];                                         // dims 64 b + 16 t .. + 15 of the row
#pragma unroll
      for (int b = 0; b < HD / 64; ++b) {
        const uint4* src = reinterpret_cast<const uint4*>(a.q + ((size_t)s * a.nh + (size_t)h * G + row) * HD + 64 * b + 16 * t);
        w[2 * b] = row < G ? src[0] : make_uint4(0, 0, 0, 0);
        w[2 * b + 1] = row < G ? src[1] : make_uint4(0, 0, 0, 0);
      }
      const uint32_t* u = reinterpret_cast<const uint32_t*>(w);
      uint32_t top = 0;                                         // the largest magnitude by its bits (an infinity or NaN is larger than any number)
#pragma unroll
      for (int i2 = 0; i2 < HD / 8; ++i2) top = max(top, max(u[i2] & 0x7fffu, (u[i2] >> 16) & 0x7fffu));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max((int)(top >> 7), 28);                   // biased exponent of the largest; tiny rows stay tiny
      const float down = __int_as_float((261 - e) << 23);       // 2^(7 - (e - 127)); e from 28 to 254
      c[r] = top >= 0x7f80u ? __int_as_float(0x7fffffff) : __int_as_float((e - 7) << 23) * a.scale * KD_LOG2E;
#pragma unroll
      for (int k = 0; k < HD / 16; ++k) {
        const float x[4] = {__uint_as_float(u[2 * k] << 16) * down, __uint_as_float(u[2 * k] & 0xffff0000u) * down,
                            __uint_as_float(u[2 * k + 1] << 16) * down, __uint_as_float(u[2 * k + 1] & 0xffff0000u) * down};
        const uint32_t p0 = kv8_codes2(x[0], x[1]), p1 = kv8_codes2(x[2], x[3]);
        const float2 y0 = kv8_float2(p0), y1 = kv8_float2(p1);
        qf[k][0][r] = p0 | p1 << 16;
        qf[k][1][r] = kv8_codes2(x[0] - y0.x, x[1] - y0.y) | kv8_codes2(x[2] - y1.x, x[3] - y1.y) << 16;
      }
      m[r] = M[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int d = 0; d < HD / 16; ++d) o[d][r][0] = o[d][r][1] = o[d][r][2] = o[d][r][3] = 0.f;
    }
  };
  // what a row's lanes (those of g) hold, for the two heads 2 t and 2 t + 1 of the thread's results
  auto of_heads = [&](float x) { return make_float2(__shfl_sync(0xffffffffu, x, 8 * t), __shfl_sync(0xffffffffu, x, 8 * t + 4)); };
  // parts of pairs: the one a warp ends with in its ring, which nothing uses any more, one that another warp began before it in global memory
  auto part_of = [&](int w, bool at_end) {
    return at_end ? reinterpret_cast<float*>(smem + w * L::SLOTS * L::TILE) : a.part + (size_t)(blockIdx.x * WARPS + w) * G * L::PART;
  };
  auto finish = [&](int i_end) {
    const int n = start[seq + 1] - start[seq], at = x0 + unit_first - start[seq] * a.nkv - kvh * n, count = i_end - unit_first;
    const bool whole = at == 0 && count == n;
    float* part = part_of(warp, i_end == n_items);
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const int row = g + 8 * r;
      float sum = l[r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      // 2^-15 o is 2^-M times sum 2^(x + E) code; times this it is the sum of 2^(x - m) 2^E code
      float f = m[r] == -INFINITY || M[r] == -INFINITY ? 0.f : kv8_ex2(M[r] - m[r]);
      if (whole) {
        const float sink = a.sinks && row < G ? a.sinks[kvh * G + row] * KD_LOG2E : -INFINITY, top = fmaxf(m[r], sink);
        const float base = top == -INFINITY ? 0.f : top, shrink = kv8_ex2(m[r] - base);
        sum = sum * shrink + kv8_ex2(sink - base);
        f = sum == 0.f ? 0.f : f * shrink / sum;
      } else if (row < G && t == 0) {
        *reinterpret_cast<float2*>(part + row * L::PART) = make_float2(m[r], sum);
      }
      const float2 fh = of_heads(f);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int head = 8 * r + 2 * t + h;
        if (head >= G) continue;
        const float fx = h ? fh.y : fh.x;
        bf16* dst = a.out + ((size_t)seq * a.nh + kvh * G + head) * HD + g;
        float* dstp = part + head * L::PART + 2 + g;
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          const float x = o[d][r][h] * KD_DOWN * fx, y = o[d][r][2 + h] * KD_DOWN * fx;
          if (whole) {
            dst[16 * d] = __float2bfloat16_rn(x);
            dst[16 * d + 8] = __float2bfloat16_rn(y);
          } else {
            dstp[16 * d] = x;
            dstp[16 * d + 8] = y;
          }
        }
      }
    }
  };

  bool ok = true;
  int done = 0;
  for (int i = -L::AHEAD; i < n_items; ++i) {
    if (((i + L::AHEAD) & 31) == 0) {                           // the next 32 items
      const int x = i + L::AHEAD + lane;
      if (x < n_items) {
        int s = seq0;
        while (start[s + 1] * a.nkv <= x0 + x) ++s;
        const int n = start[s + 1] - start[s], at = x0 + x - start[s] * a.nkv;
        const int h = at / n, j = kd_range(a, a.seq_lens[s] + a.len_add).x + at - h * n, page = a.block_table[(size_t)(a.row_seq ? a.row_seq[s] : s) * a.maxp + j];
        desc[x & (KD_DESC - 1)] = make_int4(s, h, j, (unsigned)page < (unsigned)a.n_pages ? page : 0);
      }
      __syncwarp();
      // the first tiles: half of the slots before the query is looked at, half behind it, so that a warp's first keys do not wait for all others' rings
      // (all at once: 17.4 us for 8 x 4,096 keys where this takes 16.3)
      if (i == -L::AHEAD)
#pragma unroll 1
        for (int n = 0; n < FIRST; ++n) issue(n);
    }
    if (lane < 8 && i + L::AHEAD < n_items) {                   // exponents: four lanes for the keys', four for the values'
      const int4 d = desc[(i + L::AHEAD) & (KD_DESC - 1)];
      const uint8_t* src = (lane < 4 ? a.ke : a.ve) + ((size_t)d.w * a.nkv + d.y) * SX_PAGE + 16 * t;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 16;\n" ::"r"(kd_smem(exps + ((i + L::AHEAD) & L::AHEAD) * L::EXPS + 16 * lane)), "l"(src) : "memory");
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
    if (i < 0) continue;
    done = i;
    const int4 d = desc[i & (KD_DESC - 1)];
    if (d.x != seq || d.y != kvh) {
      begin(d.x, d.y, i);
      if (i == 0) {
        unit0 = d.x * a.nkv + d.y;
#pragma unroll 1
        for (int n = FIRST; n < L::SLOTS; ++n) issue(n);
      }
    }
    const int v0 = a.window > 0 ? max(0, len - a.window - d.z * SX_PAGE) : 0, v1 = len - d.z * SX_PAGE;   // visible keys of the page: v0 <= key < v1
    const bool edge = v0 > 0 || v1 < SX_PAGE;
    // ---- scores
    int n = 2 * i, slot = n % L::SLOTS;
    ok = ok && kd_wait(bar_a + slot * 8, (n / L::SLOTS) & 1);
    if (!__all_sync(0xffffffffu, ok)) break;
    unsigned char* tile = ring + slot * L::TILE;
    float s[8][2 * RP];                                         // keys 16 t + 2 j + {0, 1}, rows g (+ 8)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned char* row = tile + (16 * (g >> 1) + 2 * j + (g & 1)) * 64 + 16 * t;
      float acc[4] = {0.f, 0.f, 0.f, 0.f}, rest[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < HD / 64; ++b) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + b * 4096);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t b0_ = h ? w.z : w.x, b1_ = h ? w.w : w.y;
          const int k = 4 * b + 2 * h;
          if (MORE) {
            kv8_mma_e4m3(acc, qf[k][0][0], qf[k][0][RP - 1], qf[k + 1][0][0], qf[k + 1][0][RP - 1], b0_, b1_);
            kv8_mma_e4m3(rest, qf[k][1][0], qf[k][1][RP - 1], qf[k + 1][1][0], qf[k + 1][1][RP - 1], b0_, b1_);
          } else {
            kv8_mma_e4m3(acc, qf[k][0][0], qf[k][1][0], qf[k + 1][0][0], qf[k + 1][1][0], b0_, b1_);
          }
        }
      }
#pragma unroll
      for (int e = 0; e < 2 * RP; ++e) s[j][e] = acc[e] + (MORE ? rest[e] : acc[2 + e]);
    }
    asm volatile("cp.async.wait_group %0;\n" ::"n"(L::AHEAD) : "memory");      // this item's are there, those of the next ones may be on their way
    __syncwarp();
    issue(n + L::SLOTS);
    const uint4 ke4 = *reinterpret_cast<const uint4*>(exps + (i & L::AHEAD) * L::EXPS + 16 * t);     // of the thread's keys 16 t ..
    const uint4 ve4 = *reinterpret_cast<const uint4*>(exps + (i & L::AHEAD) * L::EXPS + SX_PAGE + 16 * t);
    const uint32_t ke[4] = {ke4.x, ke4.y, ke4.z, ke4.w};
    float top[RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) top[r] = m[r];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // 2^(e - 127) from the byte's bits (255: an infinity, which times the NaN of such a row's codes is NaN)
        const int at = 2 * (j & 1) + e;
        const float kf = __uint_as_float((at < 3 ? ke[j >> 1] << (23 - 8 * at) : ke[j >> 1] >> 1) & 0x7f800000u);
#pragma unroll
        for (int r = 0; r < RP; ++r) s[j][2 * r + e] *= kf * c[r];
      }
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = 16 * t + 2 * j + e;
#pragma unroll
          for (int r = 0; r < RP; ++r)
            if (key < v0 || key >= v1) s[j][2 * r + e] = -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int r = 0; r < RP; ++r) top[r] = fmaxf(top[r], fmaxf(s[j][2 * r], s[j][2 * r + 1]));
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float base = top[r] == -INFINITY ? 0.f : top[r];
      float sum = l[r] * kv8_ex2(m[r] - base);
      m[r] = top[r];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += kv8_ex2(s[j][2 * r] - base) + kv8_ex2(s[j][2 * r + 1] - base);
      l[r] = sum;
    }
    // ---- weights with the values' powers of two, p v
    n = 2 * i + 1;
    slot = n % L::SLOTS;
    ok = ok && kd_wait(bar_a + slot * 8, (n / L::SLOTS) & 1);
    if (!__all_sync(0xffffffffu, ok)) break;
    tile = ring + slot * L::TILE;
    if (edge) {                                                 // codes of keys that are not seen may be anything: zeros instead
      uint32_t keep[4];                                         // bytes of the lane's 16 keys, the same in every row it has
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = ((lane & 3) << 4) + 4 * k, lo = min(max(v0 - key, 0), 4), hi = min(max(v1 - key, 0), 4);
        keep[k] = (hi == 4 ? ~0u : (1u << (8 * hi)) - 1u) & (lo == 4 ? 0u : ~((1u << (8 * lo)) - 1u));
      }
#pragma unroll 4
      for (int at = lane * 16; at < L::TILE; at += 512) {
        uint4 w = *reinterpret_cast<uint4*>(tile + at);
        w.x &= keep[0]; w.y &= keep[1]; w.z &= keep[2]; w.w &= keep[3];
        *reinterpret_cast<uint4*>(tile + at) = w;
      }
      asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");      // (the next copy into this slot comes behind these writes)
      __syncwarp();
    }
    const uint32_t ve[4] = {ve4.x, ve4.y, ve4.z, ve4.w};
    float Top[RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) Top[r] = M[r];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // the byte as the last one of 2^23 + byte.  (A row that is not finite is NaN by its codes, whatever its weight.)
        const float E = __uint_as_float(__byte_perm(ve[j >> 1], 0x4b000000u, 0x7440 + 2 * (j & 1) + e)) - 8388735.f;
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          s[j][2 * r + e] += E;
          Top[r] = fmaxf(Top[r], s[j][2 * r + e]);
        }
      }
    bool moved = false;
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      Top[r] = fmaxf(Top[r], __shfl_xor_sync(0xffffffffu, Top[r], 1));
      Top[r] = fmaxf(Top[r], __shfl_xor_sync(0xffffffffu, Top[r], 2));
      moved = moved || Top[r] != M[r];
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int r = 0; r < RP; ++r) {
        const float2 shrink = of_heads(Top[r] == -INFINITY ? 1.f : kv8_ex2(M[r] - Top[r]));
        M[r] = Top[r];
#pragma unroll
        for (int d2 = 0; d2 < HD / 16; ++d2) {
          o[d2][r][0] *= shrink.x; o[d2][r][1] *= shrink.y;
          o[d2][r][2] *= shrink.x; o[d2][r][3] *= shrink.y;
        }
      }
    }
    uint32_t p[8][RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const float base = M[r] == -INFINITY ? 0.f : M[r] - 15.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j][r] = kv8_pack2(kv8_ex2(s[j][2 * r] - base), kv8_ex2(s[j][2 * r + 1] - base));
    }
#pragma unroll
    for (int d2 = 0; d2 < HD / 16; ++d2) {
      const uint4 w0 = *reinterpret_cast<const uint4*>(tile + (16 * d2 + g) * 64 + 16 * t);
      const uint4 w1 = *reinterpret_cast<const uint4*>(tile + (16 * d2 + 8 + g) * 64 + 16 * t);
      const uint32_t u0[4] = {w0.x, w0.y, w0.z, w0.w}, u1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t a0, a1, a2, a3;
        kv8_half4(u0[k], a0, a2);
        kv8_half4(u1[k], a1, a3);
#pragma unroll
        for (int r = 0; r < RP; ++r) kv8_mma_f16(o[d2][r], a0, a1, a2, a3, p[2 * k][r], p[2 * k + 1][r]);
      }
    }
    __syncwarp();
    issue(n + L::SLOTS);
    const int4 next = desc[(i + 1) & (KD_DESC - 1)];            // (of the last item: anything)
    if (i + 1 == n_items || next.x != seq || next.y != kvh) finish(i + 1);
  }
  if (!__all_sync(0xffffffffu, ok)) {
    if (lane == 0) sx_set_status(a.status, 1);
    for (int s = 0; s < L::SLOTS; ++s) {                        // what is still under way into the slots, with a limit
      const int n = 2 * done + s;
      if ((n >> 1) < n_items) kd_wait(bar_a + n % L::SLOTS * 8, (n / L::SLOTS) & 1);
    }
  }
  // sequences without a visible key are nobody's items
  for (int s = blockIdx.x * WARPS + warp; s < a.S; s += gridDim.x * WARPS)
    if (start[s + 1] == start[s])
      for (int i = lane; i < a.nh * HD; i += 32) a.out[(size_t)s * a.nh * HD + i] = __float2bfloat16_rn(0.f);
  // ---- pairs that several warps worked at, or that go on in another block, are joined: their rows are dealt out to all warps
  const int unit1 = n_items ? seq * a.nkv + kvh : -1;
  if (lane == 0) {
    first_unit[warp] = unit0;
    last_unit[warp] = unit1;
  }
  __syncthreads();
  // lanes 0-15 look at warp k's first pair (unless a warp before has a part of it, too), lanes 16-31 at its last one where that is another
  const int k_ = lane & 15, fu = k_ < WARPS ? first_unit[k_] : -1, lu = k_ < WARPS ? last_unit[k_] : -1;
  int before = lu;
#pragma unroll
  for (int o_ = 1; o_ < 16; o_ <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before, o_, 16);
    if (k_ >= o_) before = max(before, y);
  }
  before = __shfl_up_sync(0xffffffffu, before, 1, 16);
  const int mine = lane < 16 ? fu : lu, mine_s = max(mine, 0) / a.nkv, mine_h = max(mine, 0) - mine_s * a.nkv;
  const int mine_n = start[mine_s + 1] - start[mine_s], mine_from = start[mine_s] * a.nkv + mine_h * mine_n;
  const bool met = mine < 0 || (lane < 16 ? k_ > 0 && before == fu : lu == fu);
  const bool alone = mine_from >= first_of(k_) && mine_from + mine_n <= first_of(k_ + 1);      // written by its warp
  const uint32_t joins = __ballot_sync(0xffffffffu, !met && !alone);
  int turn = warp;                                              // rows go to the warps in turn
#pragma unroll 1
  for (uint32_t left = joins; left; left &= left - 1) {
    const int from_lane = __ffs(left) - 1;
    const int u = __shfl_sync(0xffffffffu, mine, from_lane), us = __shfl_sync(0xffffffffu, mine_s, from_lane);
    const int from = __shfl_sync(0xffffffffu, mine_from, from_lane), n = __shfl_sync(0xffffffffu, mine_n, from_lane);
    const int head0 = __shfl_sync(0xffffffffu, mine_h, from_lane) * G;
    const bool final = from >= b0 && from + n <= b1, has = lane < WARPS && fu >= 0 && fu <= u && u <= lu;
    const uint32_t have = __ballot_sync(0xffffffffu, has);      // warps with a part of u
    const uint32_t inside = have & ~__ballot_sync(0xffffffffu, u == lu);       // those for whom it is not the last one
#pragma unroll 1
    for (; turn < G; turn += WARPS) {
      const int row = turn, head = head0 + row;
      float2 v[WARPS][HD / 64];
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float* src = part_of(k, !(inside >> k & 1)) + row * L::PART + 2 + 2 * lane;
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) v[k][h] = have >> k & 1 ? *reinterpret_cast<const float2*>(src + 64 * h) : make_float2(0.f, 0.f);
      }
      const float2 ml = has ? *reinterpret_cast<const float2*>(part_of(lane, u == lu) + row * L::PART) : make_float2(-INFINITY, 0.f);
      const float sink = final && a.sinks ? a.sinks[head] * KD_LOG2E : -INFINITY;
      const float top = fmaxf(warp_max(ml.x), sink), base = top == -INFINITY ? 0.f : top;
      float w = kv8_ex2(ml.x - base);
      const float sum = warp_sum(ml.y * w) + kv8_ex2(sink - base);
      if (final) w = sum == 0.f ? 0.f : __fdividef(w, sum);
      float2 x[HD / 64];
#pragma unroll
      for (int h = 0; h < HD / 64; ++h) x[h] = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float f = __shfl_sync(0xffffffffu, w, k);
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) {
          x[h].x += f * v[k][h].x;
          x[h].y += f * v[k][h].y;
        }
      }
      // a pair's first stretch goes to the block's second place, one that another block began to its first
      float* dst = a.part + ((size_t)(gridDim.x * WARPS + blockIdx.x * 2 + (from >= b0 ? 1 : 0)) * G + row) * L::PART;
      if (!final && lane == 0) *reinterpret_cast<float2*>(dst) = make_float2(top, sum);
#pragma unroll
      for (int h = 0; h < HD / 64; ++h) {
        const int d = 2 * lane + 64 * h;
        if (final) *reinterpret_cast<__nv_bfloat162*>(a.out + ((size_t)us * a.nh + head) * HD + d) = __floats2bfloat162_rn(x[h].x, x[h].y);
        else *reinterpret_cast<float2*>(dst + 2 + d) = x[h];
      }
    }
    turn -= G;
  }
}

// Pairs that several blocks shared: block b looks at the border between the stretches b and b + 1, and where that lies within a pair, takes its share of
// the pair's rows, dealt to the blocks at its borders.  With few parts a warp takes a row, with more than four the warps share a row's parts.  Lengths are
// read and the place is found while the first kernel still runs: it lets this one in behind its own wait, so what was there before it is there.
// (As a block of 256 threads for every border and row: 29.7 us for 64 sequences seeing 1,000 keys where this took 27.3, 18.3 for 8 x 4,096 where it took
// 17.3.  Fewer registers in the first kernel, so that these blocks wait on its SMs, cost it more than that gave: 18.8 for 8 x 4,096, 56.6 for one of 131,072
// where 52.8 stood.)
#define KD_MERGE_WARPS 4
template <int HD>
__global__ void __launch_bounds__(KD_MERGE_WARPS * 32) kv8_decode_merge_kernel(const KdArgs a) {
  constexpr int DIMS = HD / 32, TEAMS = KD_MERGE_WARPS;         // dims a lane
  extern __shared__ int start[];
  __shared__ int warp_sums[TEAMS];
  __shared__ float acc[TEAMS][HD], s_m[TEAMS], s_l[TEAMS];
  kd_starts<TEAMS * 32>(a, start, warp_sums);
  const int G = a.nh / a.nkv, n_all = start[a.S] * a.nkv, workers = n_all ? kd_workers(a, n_all) : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int w0 = 0, k = 0, seq = 0, kvh = 0;                          // the pair's first block, and the borders within the pair
  if ((int)blockIdx.x + 1 < workers) {
    const int border = kd_first(blockIdx.x + 1, n_all, workers);
    seq = kd_seq_of(start, a.S, a.nkv, border);
    const int n = start[seq + 1] - start[seq], at = border - start[seq] * a.nkv;
    kvh = at / n;
    const int from = start[seq] * a.nkv + kvh * n;
    if (from < border) {
      w0 = kd_worker_of(from, n_all, workers);
      k = kd_worker_of(from + n - 1, n_all, workers) - w0;
    }
  }
  pdl_wait();
  pdl_trigger();
  if (k == 0) return;
  const bool shared = k >= TEAMS;                               // (of the pair, so of the block)
  const int team = shared ? warp : 0, teams = shared ? TEAMS : 1, rows = shared ? 1 : TEAMS, step = 2 * G * (HD + 2);
  for (int row0 = ((int)blockIdx.x - w0) * rows; row0 < G; row0 += k * rows) {
    const int row = shared ? row0 : row0 + warp, head = kvh * G + row;
    if (row >= G) break;                                        // (never where a row is shared)
    // (blocks at work are never more than items, so every one from w0 to w0 + k has a part; the first block's is in its second place)
    const float* parts = a.part + ((size_t)(a.blocks * a.warps + 2 * w0) * G + row) * (HD + 2);
    const float sink = a.sinks ? a.sinks[head] * KD_LOG2E : -INFINITY;
    float top = -INFINITY, L = 0.f, x[DIMS] = {};
    for (int w = team; w <= k; w += 4 * teams) {
      float2 ml[4], v[4][DIMS / 2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = w + j * teams;
        ml[j] = make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int d = 0; d < DIMS / 2; ++d) v[j][d] = make_float2(0.f, 0.f);
        if (i <= k) {
          const float2* src = reinterpret_cast<const float2*>(parts + (ptrdiff_t)i * step + (i == 0 ? step / 2 : 0));
          ml[j] = src[0];
#pragma unroll
          for (int d = 0; d < DIMS / 2; ++d) v[j][d] = src[1 + d * 32 + lane];
        }
      }
      const float next = fmaxf(fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x)), top), base = next == -INFINITY ? 0.f : next;
      const float f = kv8_ex2(top - base);
      L *= f;
#pragma unroll
      for (int d = 0; d < DIMS; ++d) x[d] *= f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float h = kv8_ex2(ml[j].x - base);
        L += ml[j].y * h;
#pragma unroll
        for (int d = 0; d < DIMS / 2; ++d) {
          x[2 * d] += v[j][d].x * h;
          x[2 * d + 1] += v[j][d].y * h;
        }
      }
      top = next;
    }
    bf16* dst = a.out + ((size_t)seq * a.nh + head) * HD;
    if (!shared) {
      const float all = fmaxf(top, sink), base = all == -INFINITY ? 0.f : all, f = kv8_ex2(top - base);
      L = L * f + kv8_ex2(sink - base);
      const float inv = L == 0.f ? 0.f : f / L;
#pragma unroll
      for (int d = 0; d < DIMS / 2; ++d) reinterpret_cast<__nv_bfloat162*>(dst)[d * 32 + lane] = __floats2bfloat162_rn(x[2 * d] * inv, x[2 * d + 1] * inv);
      continue;
    }
#pragma unroll
    for (int d = 0; d < DIMS / 2; ++d) reinterpret_cast<float2*>(acc[team])[d * 32 + lane] = make_float2(x[2 * d], x[2 * d + 1]);
    if (lane == 0) {
      s_m[team] = top;
      s_l[team] = L;
    }
    __syncthreads();
    if (threadIdx.x < HD) {
      float all = sink;
#pragma unroll
      for (int i = 0; i < TEAMS; ++i) all = fmaxf(all, s_m[i]);
      const float base = all == -INFINITY ? 0.f : all;
      float den = kv8_ex2(sink - base), O = 0.f;
#pragma unroll
      for (int i = 0; i < TEAMS; ++i) {
        const float f = kv8_ex2(s_m[i] - base);
        den += s_l[i] * f;
        O += acc[i][threadIdx.x] * f;
      }
      dst[threadIdx.x] = __float2bfloat16_rn(den == 0.f ? 0.f : O / den);
    }
    __syncthreads();
  }
}

static int* kd_status() {
  static int* word = sx_status_word_alloc();
  return word;
}
extern "C" int sx_kv8_decode_status(int* value, int reset) {
  int* w = kd_status();
  if (!w) return SX_ERR_SIZE;
  *value = *(volatile int*)w;
  if (reset) *w = 0;
  return 0;
}

template <int HD, bool MORE>
static int kd_launch(KdArgs a, cudaStream_t stream) {
  using L = KdLayout<HD, MORE>;
  static bool opted[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64 || !opted[dev]) {
    e = cudaFuncSetAttribute(kv8_decode_kernel<HD, MORE>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::FIXED + KD_MAX_SEQS * (int)sizeof(int));
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) opted[dev] = true;
  }
  a.warps = L::WARPS;
  const int rc = sx_launch(kv8_decode_kernel<HD, MORE>, dim3(a.blocks), dim3(L::WARPS * 32), L::FIXED + (a.S <= KD_FEW_SEQS ? L::WARPS : 1) * (a.S + 1) * sizeof(int), stream, a);
  if (rc || a.by_pair || a.blocks == 1) return rc;
  return sx_launch(kv8_decode_merge_kernel<HD>, dim3(a.blocks - 1), dim3(KD_MERGE_WARPS * 32), (a.S + 1) * sizeof(int), stream, a);
}

// a block a pair: pairs no more than SMs, of no more than two pages a warp
static bool kd_by_pair(int S, int nkv, int max_pages) { return (long long)S * nkv <= sx_sm_count() && max_pages <= 24; }
static int kd_blocks(int S, int nkv, int max_pages) {
  const long long items = (long long)S * nkv * max_pages, few = (items + 7) / 8;         // (the fewest warps of a block are 8)
  return kd_by_pair(S, nkv, max_pages) ? S * nkv : (int)max(1ll, min((long long)sx_sm_count(), few));
}
// kernels that a launch makes, and floats of `part` it needs
extern "C" int sx_kv8_decode_plan(int S, int nh, int nkv, int hd, int max_pages, long long* floats) {
  *floats = 0;
  if (nkv <= 0) return 0;
  if (kd_by_pair(S, nkv, max_pages)) return 1;                  // (a warp's only part is in shared memory)
  const int blocks = kd_blocks(S, nkv, max_pages);
  *floats = (long long)blocks * (KD_MAX_WARPS + 2) * (nh / nkv) * (hd + 2);
  return blocks == 1 ? 1 : 2;
}

// A row of q is a sequence's only token (row_seq null, len_add 0), or any token: seq_lens then holds positions, len_add is 1 and row_seq says whose
// table it reads.  max_pages: no row has more visible pages
extern "C" int sx_kv8_decode(const void* q, void* out, const void* k, const void* v, const void* k_exp, const void* v_exp, const int* seq_lens,
                             const int* row_seq, int len_add, const int* block_table, int maxp, int S, int nh, int nkv, int hd, int n_pages, float scale, int window,
                             const float* sinks, float* part, int max_pages, cudaStream_t stream) {
  if (S <= 0) return 0;
  if ((hd != 64 && hd != 128) || nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > 16 || S >= KD_MAX_SEQS || n_pages <= 0 || maxp <= 0 || max_pages <= 0 ||
      (long long)S * nkv * maxp >= (1ll << 31) || (long long)S * nh >= (1ll << 31) || (!part && !kd_by_pair(S, nkv, max_pages)))
    return SX_ERR_SIZE;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_exp | (uintptr_t)v_exp | (uintptr_t)part) & 15) return SX_ERR_ALIGN;
  int* status = kd_status();
  if (!status) return SX_ERR_SIZE;
  const KdArgs a = {(const bf16*)q, (bf16*)out, (const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_exp, (const uint8_t*)v_exp, seq_lens, row_seq, block_table,
                    sinks, part, status, len_add, maxp, n_pages, S, nh, nkv, window, kd_blocks(S, nkv, max_pages), 0, kd_by_pair(S, nkv, max_pages), scale};
  if (hd == 64) return nh / nkv > 8 ? kd_launch<64, true>(a, stream) : kd_launch<64, false>(a, stream);
  return nh / nkv > 8 ? kd_launch<128, true>(a, stream) : kd_launch<128, false>(a, stream);
}
