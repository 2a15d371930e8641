// Attention of single tokens over a cache in eight bits (kv8.cuh) on the tensor cores: bfloat16 queries, head size 64 or 128, up to 16
// query heads a kv head.
//
// A single token reads every code once, so the kernel has to keep HBM busy: 16.1 KB a page and kv head at head size 128 against
// 0.5 M operations.  Everything is done by warps on their own:
//   * The visible pages of all (sequence, kv head) pairs are one line of items, and each warp takes an equal stretch of it, whatever
//     the sequences' lengths are; a pair that several warps share is joined by a second, small kernel.
//   * A warp has its own ring of shared memory, filled by untiled bulk copies (K and V tile of a page are one stretch of memory each;
//     no tensor map), and no barrier with other warps.  K and V take turns in the slots, so a slot is free again after half a page.
//   * q k^T: the G heads are the M rows of m16n8k16 in half precision.  e4m3 codes become half precision exactly (one conversion for two),
//     queries are bfloat16 scaled by a power of two of the row's so that its largest lies in 2^14 .. 2^15: every element down to 2^-28 of
//     that is exact too.  The order of the inner axis is free as long as both operands agree, so a thread takes 16 neighbouring codes
//     of a key in one 16-byte load (four k-steps' worth) and the query's elements to match.
//   * The same freedom in p v (values lie dim by dim): with keys dealt to columns as 16 t + 2 j + i, the scores a thread holds are exactly
//     the weights its fragments need, and the exponents of its 16 keys are one 16-byte load.  Nothing moves between lanes but the
//     row's maxima.
//   * A value's power of two joins the weight before it is rounded: with x the score (base 2) and E the exponent, weights are 2^(x - m) in
//     the denominator, and 2^(x + E - M + 15) in half precision beside the codes, with M the running maximum of x + E.  So a large value
//     of next to no weight takes nothing from the precision of the others; weights from 1 down to 2^-29 of the row's largest x + E keep all 11 bits.
//
// Every wait on an mbarrier is bounded; one that runs out sets the library's status word (sx_kv8_decode_status).
#include "kv8.cuh"

#define KD_WARPS 8
#define KD_MAX_SEQS 2048
#define KD_SPIN_LIMIT (1u << 26)
#define KD_DOWN 3.0517578125e-5f      // 2^-15
#define KD_DESC 64               // items a warp knows ahead: two batches of 32

template <int HD> struct KdLayout {
  static constexpr int TILE = SX_PAGE * HD;
  static constexpr int SLOT = TILE + 128;                       // a K or V tile and its 64 exponents
  static constexpr int SLOTS = HD == 128 ? 3 : 6;
  static constexpr int RING = KD_WARPS * SLOTS * SLOT;
  static constexpr int smem() { return RING + KD_WARPS * KD_DESC * (int)sizeof(int4) + KD_MAX_SEQS * (int)sizeof(int) + 128; }
};

struct KdArgs {
  const bf16* q;
  bf16* out;
  const uint8_t *k, *v, *ke, *ve;
  const int *seq_lens, *block_table;
  const float* sinks;
  float* part;                 // [warps][2][rows of a kv head][HD + 2]
  int* status;
  int maxp, n_pages, S, nh, nkv, window, warps, min_pages;
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
__device__ __forceinline__ void kd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float kd_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t kd_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// first visible page of a sequence and one behind its last
__device__ __forceinline__ int2 kd_range(const KdArgs& a, int s) {
  const int len = a.seq_lens[s];
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
      const int2 r = kd_range(a, s);
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
// the warps that work and the first item of warp w (of all items `n`)
__device__ __forceinline__ int kd_workers(const KdArgs& a, int n) { return max(1, min(a.warps, (n + a.min_pages - 1) / a.min_pages)); }
__device__ __forceinline__ int kd_first(int w, int n, int workers) { return (int)((long long)w * n / workers); }
__device__ __forceinline__ int kd_worker_of(int item, int n, int workers) { return (int)((((long long)item + 1) * workers - 1) / n); }
// the sequence of item x: the last s with start[s] * nkv <= x among those that have pages
__device__ __forceinline__ int kd_seq_of(const int* start, int S, int nkv, int x) {
  int lo = 0, hi = S - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] * nkv <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// MORE: more than 8 query heads a kv head, so that the fragments' second eight rows are used
template <int HD, bool MORE>
__global__ void __launch_bounds__(KD_WARPS * 32, 1) kv8_decode_kernel(const KdArgs a) {
  using L = KdLayout<HD>;
  constexpr int RP = MORE ? 2 : 1;                              // rows a thread has
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ __align__(8) uint64_t bars[KD_WARPS * L::SLOTS];
  __shared__ int warp_sums[KD_WARPS];
  int4* desc_all = reinterpret_cast<int4*>(smem + L::RING);
  int* start = reinterpret_cast<int*>(smem + L::RING + KD_WARPS * KD_DESC * sizeof(int4));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (lane == 0) {
#pragma unroll
    for (int s = 0; s < L::SLOTS; ++s) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;\n" ::"r"(kd_smem(&bars[warp * L::SLOTS + s])));
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
  }
  pdl_wait();
  pdl_trigger();
  kd_starts<KD_WARPS * 32>(a, start, warp_sums);
  const int G = a.nh / a.nkv, n_all = start[a.S] * a.nkv;
  const int workers = kd_workers(a, n_all), me = warp * gridDim.x + blockIdx.x;      // neighbours on different SMs
  if (n_all == 0) {                                             // nobody sees anything
    for (size_t i = blockIdx.x * KD_WARPS * 32 + threadIdx.x; i < (size_t)a.S * a.nh * HD; i += gridDim.x * KD_WARPS * 32) a.out[i] = __float2bfloat16_rn(0.f);
    return;
  }
  // sequences without a visible key are nobody's items
  for (int s = me; s < a.S; s += gridDim.x * KD_WARPS)
    if (start[s + 1] == start[s])
      for (int i = lane; i < a.nh * HD; i += 32) a.out[(size_t)s * a.nh * HD + i] = __float2bfloat16_rn(0.f);
  if (me >= workers) return;
  const int x0 = kd_first(me, n_all, workers), n_items = kd_first(me + 1, n_all, workers) - x0;
  int4* desc = desc_all + warp * KD_DESC;                       // (sequence, kv head, page of the sequence, page of the pool)
  auto describe = [&](int batch) {
    const int i = batch * 32 + lane;
    if (i < n_items) {
      const int s = kd_seq_of(start, a.S, a.nkv, x0 + i), n = start[s + 1] - start[s], at = x0 + i - start[s] * a.nkv;
      const int kvh = at / n, j = kd_range(a, s).x + at % n, page = a.block_table[(size_t)s * a.maxp + j];
      desc[i & (KD_DESC - 1)] = make_int4(s, kvh, j, (unsigned)page < (unsigned)a.n_pages ? page : 0);
    }
    __syncwarp();
  };
  unsigned char* ring = smem + warp * L::SLOTS * L::SLOT;
  const uint32_t ring_a = kd_smem(ring), bar_a = kd_smem(&bars[warp * L::SLOTS]);
  // load number n of the warp: the K (even) or V (odd) tile of item n / 2, into slot n % SLOTS
  auto issue = [&](int n) {
    const int i = n >> 1;
    if (i >= n_items) return;
    if (!(n & 1) && (i & 31) == 0) describe(i >> 5);
    if (lane == 0) {
      const int4 d = desc[i & (KD_DESC - 1)];
      const size_t place = (size_t)d.w * a.nkv + d.y;
      const int slot = n % L::SLOTS;
      const uint32_t dst = ring_a + slot * L::SLOT, bar = bar_a + slot * 8;
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"(L::TILE + SX_PAGE) : "memory");
      kd_copy(dst, ((n & 1) ? a.v : a.k) + place * L::TILE, L::TILE, bar);
      kd_copy(dst + L::TILE, ((n & 1) ? a.ve : a.ke) + place * SX_PAGE, SX_PAGE, bar);
    }
  };
#pragma unroll
  for (int n = 0; n < L::SLOTS; ++n) issue(n);

  uint32_t qf[HD / 16][2 * RP];
  float c[RP], m[RP], l[RP], M[RP], o[HD / 8][4];
  int seq = -1, kvh = -1, unit_first = 0;                       // the pair at work and the item of the warp it began with
  auto begin = [&](int s, int h, int i) {
    seq = s; kvh = h; unit_first = i;
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const int row = g + 8 * r;
      uint4 w[HD / 32];                                         // dims 64 c + 16 t .. + 15 of the row
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
      const float down = __int_as_float((268 - e) << 23);       // 2^(14 - (e - 127)); e from 28 to 254
      c[r] = top >= 0x7f80u ? __int_as_float(0x7fffffff) : __int_as_float(max(e - 14, 1) << 23) * a.scale * 1.44269504f;
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
#pragma unroll
        for (int h2 = 0; h2 < 2; ++h2) {
          const uint32_t pair = u[(ks >> 2) * 8 + (ks & 3) * 2 + h2];
          qf[ks][h2 * RP + r] = kd_half2(__uint_as_float(pair << 16) * down, __uint_as_float(pair & 0xffff0000u) * down);
        }
      m[r] = M[r] = -INFINITY;
      l[r] = 0.f;
    }
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  };
  auto finish = [&](int i_end) {
    const int n = start[seq + 1] - start[seq], at = x0 + unit_first - start[seq] * a.nkv - kvh * n, count = i_end - unit_first;
    const bool whole = at == 0 && count == n;
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const int row = g + 8 * r;
      float L_ = l[r];
      L_ += __shfl_xor_sync(0xffffffffu, L_, 1);
      L_ += __shfl_xor_sync(0xffffffffu, L_, 2);
      // 2^-15 o is 2^-M times sum 2^(x + E) code; times this it is the sum of 2^(x - m) 2^E code
      float f = m[r] == -INFINITY || M[r] == -INFINITY ? 0.f : kd_ex2(M[r] - m[r]);
      if (row >= G) continue;
      const int head = kvh * G + row;
      if (whole) {
        if (a.sinks) {
          const float sink = a.sinks[head] * 1.44269504f, top = fmaxf(m[r], sink);
          const float shrink = kd_ex2(m[r] - top);
          L_ = L_ * shrink + kd_ex2(sink - top);
          f *= shrink;
        }
        f = L_ == 0.f ? 0.f : f / L_;
        bf16* dst = a.out + ((size_t)seq * a.nh + head) * HD + 2 * t;
#pragma unroll
        for (int d = 0; d < HD / 8; ++d)
          *reinterpret_cast<__nv_bfloat162*>(dst + 8 * d) = __floats2bfloat162_rn(o[d][2 * r] * KD_DOWN * f, o[d][2 * r + 1] * KD_DOWN * f);
      } else {
        // a pair's first stretch goes to the warp's second place, one that another warp began to its first
        float* dst = a.part + ((size_t)(me * 2 + (at == 0 ? 1 : 0)) * G + row) * (HD + 2);
        if (t == 0) *reinterpret_cast<float2*>(dst) = make_float2(m[r], L_);
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(dst + 2 + 8 * d + 2 * t) = make_float2(o[d][2 * r] * KD_DOWN * f, o[d][2 * r + 1] * KD_DOWN * f);
      }
    }
  };

  bool ok = true;
  int done = 0;
  for (int i = 0; i < n_items; ++i) {
    done = i;
    const int4 d = desc[i & (KD_DESC - 1)];
    if (d.x != seq || d.y != kvh) {
      if (seq >= 0) finish(i);
      begin(d.x, d.y, i);
    }
    const int len = a.seq_lens[seq];
    const int v0 = a.window > 0 ? max(0, len - a.window - d.z * SX_PAGE) : 0, v1 = len - d.z * SX_PAGE;   // visible keys of the page: v0 <= key < v1
    const bool edge = v0 > 0 || v1 < SX_PAGE;
    // ---- scores
    int n = 2 * i, slot = n % L::SLOTS;
    ok = ok && kd_wait(bar_a + slot * 8, (n / L::SLOTS) & 1);
    if (!__all_sync(0xffffffffu, ok)) break;
    const unsigned char* tile = ring + slot * L::SLOT;
    float s[8][4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
      const int key = 16 * (g >> 1) + 2 * j + (g & 1);
#pragma unroll
      for (int b = 0; b < HD / 64; ++b) {
        const uint4 w = *reinterpret_cast<const uint4*>(tile + b * 4096 + key * 64 + 16 * t);
        const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t(&qa)[2 * RP] = qf[4 * b + k];
          kd_mma(s[j], qa[0], MORE ? qa[RP - 1] : 0u, qa[RP], MORE ? qa[2 * RP - 1] : 0u, kv8_half2(ww[k]), kv8_half2(ww[k] >> 16));
        }
      }
    }
    const uint4 ke4 = *reinterpret_cast<const uint4*>(tile + L::TILE + 16 * t);    // exponents of the thread's keys 16 t ..
    __syncwarp();
    issue(n + L::SLOTS);
    const uint32_t ke[4] = {ke4.x, ke4.y, ke4.z, ke4.w};
    float top[RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) top[r] = m[r];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float kf = kv8_scale((ke[j >> 1] >> (16 * (j & 1) + 8 * e)) & 0xff);
        const int key = 16 * t + 2 * j + e;
#pragma unroll
        for (int r = 0; r < RP; ++r) {
          float x = s[j][2 * r + e] * kf * c[r];
          if (edge && (key < v0 || key >= v1)) x = -INFINITY;
          s[j][2 * r + e] = x;
          top[r] = fmaxf(top[r], x);
        }
      }
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float base = top[r] == -INFINITY ? 0.f : top[r];
      float sum = l[r] * kd_ex2(m[r] - base);
      m[r] = top[r];
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += kd_ex2(s[j][2 * r] - base) + kd_ex2(s[j][2 * r + 1] - base);
      l[r] = sum;
    }
    // ---- weights with the values' powers of two, p v
    n = 2 * i + 1;
    slot = n % L::SLOTS;
    ok = ok && kd_wait(bar_a + slot * 8, (n / L::SLOTS) & 1);
    if (!__all_sync(0xffffffffu, ok)) break;
    tile = ring + slot * L::SLOT;
    const uint4 ve4 = *reinterpret_cast<const uint4*>(tile + L::TILE + 16 * t);
    const uint32_t ve[4] = {ve4.x, ve4.y, ve4.z, ve4.w};
    float Top[RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) Top[r] = M[r];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int b = (ve[j >> 1] >> (16 * (j & 1) + 8 * e)) & 0xff, key = 16 * t + 2 * j + e;
        float E = b == KV8_NAN ? __int_as_float(0x7fffffff) : (float)(b - 127);
        if (edge && (key < v0 || key >= v1)) E = 0.f;
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
        const float shrink = Top[r] == -INFINITY ? 1.f : kd_ex2(M[r] - Top[r]);
        M[r] = Top[r];
#pragma unroll
        for (int d2 = 0; d2 < HD / 8; ++d2) {
          o[d2][2 * r] *= shrink;
          o[d2][2 * r + 1] *= shrink;
        }
      }
    }
    uint32_t p[8][RP];
#pragma unroll
    for (int r = 0; r < RP; ++r) {
      const float base = M[r] == -INFINITY ? 0.f : M[r] - 15.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) p[j][r] = kd_half2(kd_ex2(s[j][2 * r] - base), kd_ex2(s[j][2 * r + 1] - base));
    }
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};                    // codes of keys that are not seen may be anything: zeros instead
    if (edge) {
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (16 * t + k < v0 || 16 * t + k >= v1) keep[k >> 2] &= ~(0xffu << (8 * (k & 3)));
    }
#pragma unroll
    for (int d2 = 0; d2 < HD / 8; ++d2) {
      const uint4 w = *reinterpret_cast<const uint4*>(tile + (8 * d2 + g) * 64 + 16 * t);
      const uint32_t ww[4] = {w.x & keep[0], w.y & keep[1], w.z & keep[2], w.w & keep[3]};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        kd_mma(o[d2], p[2 * k][0], MORE ? p[2 * k][RP - 1] : 0u, p[2 * k + 1][0], MORE ? p[2 * k + 1][RP - 1] : 0u, kv8_half2(ww[k]),
               kv8_half2(ww[k] >> 16));
    }
    __syncwarp();
    issue(n + L::SLOTS);
    if (i + 1 == n_items) finish(n_items);
  }
  if (!__all_sync(0xffffffffu, ok)) {
    if (lane == 0) sx_set_status(a.status, 1);
    for (int s = 0; s < L::SLOTS; ++s) {                        // what is still under way into the slots, with a limit
      const int n = 2 * done + s;
      if ((n >> 1) < n_items) kd_wait(bar_a + n % L::SLOTS * 8, (n / L::SLOTS) & 1);
    }
  }
}

// Pairs that several warps shared: a block a (pair, row), 4 threads a group of dims take turns over the shares.
template <int HD>
__global__ void __launch_bounds__(256) kv8_decode_merge_kernel(const KdArgs a) {
  __shared__ int start[KD_MAX_SEQS + 1], warp_sums[8];
  __shared__ float acc[256 / (HD / 2)][HD], s_m[256 / (HD / 2)], s_l[256 / (HD / 2)];
  pdl_wait();
  pdl_trigger();
  kd_starts<256>(a, start, warp_sums);
  constexpr int TEAMS = 256 / (HD / 2);
  const int G = a.nh / a.nkv, seq = blockIdx.x / a.nh, head = blockIdx.x % a.nh, kvh = head / G, row = head % G;
  const int n = start[seq + 1] - start[seq], n_all = start[a.S] * a.nkv;
  if (n == 0) return;
  const int workers = kd_workers(a, n_all), first = start[seq] * a.nkv + kvh * n;
  const int w0 = kd_worker_of(first, n_all, workers), w1 = kd_worker_of(first + n - 1, n_all, workers);
  if (w0 == w1) return;
  const int team = threadIdx.x / (HD / 2), d = threadIdx.x % (HD / 2) * 2;
  float top = -INFINITY, L = 0.f, x = 0.f, y = 0.f;
  // (workers are never more than items, so every warp from w0 to w1 has a share)
#pragma unroll 4
  for (int w = w0 + team; w <= w1; w += TEAMS) {
    const float* src = a.part + ((size_t)(w * 2 + (w == w0 ? 1 : 0)) * G + row) * (HD + 2);
    const float2 ml = *reinterpret_cast<const float2*>(src), v = *reinterpret_cast<const float2*>(src + 2 + d);
    const float next = fmaxf(top, ml.x), base = next == -INFINITY ? 0.f : next, f = kd_ex2(top - base), h = kd_ex2(ml.x - base);
    L = L * f + ml.y * h;
    x = x * f + v.x * h;
    y = y * f + v.y * h;
    top = next;
  }
  acc[team][d] = x;
  acc[team][d + 1] = y;
  if (d == 0) {
    s_m[team] = top;
    s_l[team] = L;
  }
  __syncthreads();
  if (threadIdx.x >= HD) return;
  const float sink = a.sinks ? a.sinks[head] * 1.44269504f : -INFINITY;
  top = sink;
#pragma unroll
  for (int i = 0; i < TEAMS; ++i) top = fmaxf(top, s_m[i]);
  const float base = top == -INFINITY ? 0.f : top;
  L = a.sinks ? kd_ex2(sink - base) : 0.f;
  float O = 0.f;
#pragma unroll
  for (int i = 0; i < TEAMS; ++i) {
    const float f = kd_ex2(s_m[i] - base);
    L += s_l[i] * f;
    O += acc[i][threadIdx.x] * f;
  }
  a.out[((size_t)seq * a.nh + head) * HD + threadIdx.x] = __float2bfloat16_rn(L == 0.f ? 0.f : O / L);
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

// floats of `part` for a launch on the current device
extern "C" long long sx_kv8_decode_scratch(int nh, int nkv, int hd) {
  return (long long)sx_sm_count() * KD_WARPS * 2 * (nh / nkv) * (hd + 2);
}

template <int HD, bool MORE>
static int kd_launch(const KdArgs& a, int blocks, cudaStream_t stream) {
  static bool opted[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64 || !opted[dev]) {
    e = cudaFuncSetAttribute(kv8_decode_kernel<HD, MORE>, cudaFuncAttributeMaxDynamicSharedMemorySize, KdLayout<HD>::smem());
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) opted[dev] = true;
  }
  const int rc = sx_launch(kv8_decode_kernel<HD, MORE>, dim3(blocks), dim3(KD_WARPS * 32), KdLayout<HD>::smem(), stream, a);
  if (rc) return rc;
  return sx_launch(kv8_decode_merge_kernel<HD>, dim3(a.S * a.nh), dim3(256), 0, stream, a);
}

extern "C" int sx_kv8_decode(const void* q, void* out, const void* k, const void* v, const void* k_exp, const void* v_exp, const int* seq_lens,
                             const int* block_table, int maxp, int S, int nh, int nkv, int hd, int n_pages, float scale, int window,
                             const float* sinks, float* part, int max_pages, int min_pages, cudaStream_t stream) {
  if (S <= 0) return 0;
  if ((hd != 64 && hd != 128) || nkv <= 0 || nh <= 0 || nh % nkv || nh / nkv > 16 || S >= KD_MAX_SEQS || n_pages <= 0 || maxp <= 0 || min_pages <= 0 ||
      (long long)S * nkv * maxp >= (1ll << 31) || (long long)S * nh >= (1ll << 31) || !part)
    return SX_ERR_SIZE;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_exp | (uintptr_t)v_exp | (uintptr_t)part) & 15) return SX_ERR_ALIGN;
  int* status = kd_status();
  if (!status) return SX_ERR_SIZE;
  const long long items = (long long)S * nkv * max_pages;
  const int blocks = (int)max(1ll, min((long long)sx_sm_count(), items));
  const KdArgs a = {(const bf16*)q, (bf16*)out, (const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_exp, (const uint8_t*)v_exp, seq_lens, block_table,
                    sinks, part, status, maxp, n_pages, S, nh, nkv, window, blocks * KD_WARPS, min_pages, scale};
  if (hd == 64) return nh / nkv > 8 ? kd_launch<64, true>(a, blocks, stream) : kd_launch<64, false>(a, blocks, stream);
  return nh / nkv > 8 ? kd_launch<128, true>(a, blocks, stream) : kd_launch<128, false>(a, blocks, stream);
}
