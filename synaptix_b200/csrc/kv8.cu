// A cache of keys and values in eight bits: heads are prepared and quantised as they are written, pages are read back, and
// single tokens attend over them whatever the head size, type and options (kv8.cuh says what the format is and why).
#include "kv8.cuh"

#define KV8_MAX_HD 256

// ---------------------------------------------------------------------------------------
// Head preparation with the write into the cache.  A block a token (and a share of its heads), a warp a head:
//   q heads: x / rms(x) * gain (optional), rotate-half rotation of the first rotary_dim elements (optional), to q_out;
//   k heads: the same, then quantised into the sequence's page;   v heads: quantised.
// The rotation's angle is position * inv_freq in about 48 bits: the product rounded to 32 bits and what that left out, by which
// sine and cosine are moved on.  (In 32 bits alone an angle at position 100,000 is off by up to 0.004.)
// One token of 48 heads of 128 3.7 us, 48 tokens 4.8: a launch, the page's number from the table, a row, its sums.
// ---------------------------------------------------------------------------------------
#define KV8_WARPS 8
// cosine and sine of pos * f: the angle is hi + lo with |lo| <= 2^-24 |hi|, up to 2^-8 at position 131,072, so the series in lo needs its
// second term (lo^2 / 2 = 8e-6 there) and not its third (1e-8)
__device__ __forceinline__ float2 kv8_turn(int pos, float f) {
  const float p = (float)pos, hi = p * f, lo = fmaf(p, f, -hi), q = -0.5f * lo * lo;
  float sn, cs;
  sincosf(hi, &sn, &cs);
  return make_float2(fmaf(-lo, sn, fmaf(q, cs, cs)), fmaf(lo, cs, fmaf(q, sn, sn)));
}
template <typename T>
__global__ void __launch_bounds__(KV8_WARPS * 32) kv8_prepare_kernel(
    const T* __restrict__ qkv, T* __restrict__ q_out, uint8_t* __restrict__ k_pages, uint8_t* __restrict__ v_pages,
    uint8_t* __restrict__ k_exp, uint8_t* __restrict__ v_exp, const float* __restrict__ wq, const float* __restrict__ wk,
    const float* __restrict__ inv_freq, int rotary_dim, float eps, const int* __restrict__ positions,
    const int* __restrict__ seq_of_token, const int* __restrict__ block_table, int maxp, int nh, int nkv, int hd, int n_pages,
    int row) {
  __shared__ float s_cs[KV8_MAX_HD / 2], s_sn[KV8_MAX_HD / 2];
  __shared__ float s_x[KV8_WARPS][KV8_MAX_HD];
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = positions[t], half = inv_freq ? rotary_dim / 2 : 0;
  for (int i = threadIdx.x; i < half; i += KV8_WARPS * 32) {
    const float2 r = kv8_turn(pos, inv_freq[i]);
    s_cs[i] = r.x;
    s_sn[i] = r.y;
  }
  const int page = (unsigned)(pos >> 6) < (unsigned)maxp ? block_table[(size_t)seq_of_token[t] * maxp + (pos >> 6)] : -1;
  const bool page_ok = k_pages && page >= 0 && page < n_pages;        // the host guarantees a page; never write outside
  __syncthreads();
  const int cb = kv8_block(hd), heads = k_pages ? nh + 2 * nkv : nh;
  float* xs = s_x[warp];
  for (int head = blockIdx.y * KV8_WARPS + warp; head < heads; head += gridDim.y * KV8_WARPS) {
    const bool is_q = head < nh, is_k = !is_q && head < nh + nkv;
    const T* src = qkv + (size_t)t * row + (size_t)head * hd;
    const float* gain = is_q ? wq : is_k ? wk : nullptr;
    __syncwarp();
    float ss = 0.f;
    for (int i = lane; i < hd; i += 32) {
      const float x = to_f32(src[i]);
      xs[i] = x;
      ss += x * x;
    }
    const float inv = gain ? rsqrtf(warp_sum(ss) / (float)hd + eps) : 1.f;
    __syncwarp();
    float y[KV8_MAX_HD / 32];
    float a = 0.f;
    bool finite = true;
#pragma unroll
    for (int k = 0; k < KV8_MAX_HD / 32; ++k) {
      const int i = lane + 32 * k;
      y[k] = 0.f;
      if (i < hd) {
        float x = xs[i] * inv;
        if (gain) x *= gain[i];
        if ((is_q || is_k) && i < 2 * half) {
          const int j = i < half ? i + half : i - half, p = i < half ? i : j;
          float z = xs[j] * inv;
          if (gain) z *= gain[j];
          x = i < half ? x * s_cs[p] - z * s_sn[p] : x * s_cs[p] + z * s_sn[p];
        }
        y[k] = x;
        a = fmaxf(a, fabsf(x));
        finite = finite && fabsf(x) < INFINITY;                        // (false for NaN)
      }
    }
    if (is_q) {
      for (int k = 0; k < KV8_MAX_HD / 32; ++k)
        if (lane + 32 * k < hd) q_out[((size_t)t * nh + head) * hd + lane + 32 * k] = from_f32<T>(y[k]);
      continue;
    }
    const int e = kv8_exponent(warp_max(a), __all_sync(0xffffffffu, finite));
    if (!page_ok) continue;
    const float inverse = kv8_inverse(e);
    const int kvh = is_k ? head - nh : head - nh - nkv, key = pos & (SX_PAGE - 1);
    const size_t place = (size_t)page * nkv + kvh;
    uint8_t* dst = (is_k ? k_pages : v_pages) + place * SX_PAGE * hd;
#pragma unroll
    for (int k = 0; k < KV8_MAX_HD / 32; ++k) {
      const int i = lane + 32 * k;
      if (i < hd) dst[is_k ? kv8_k_at(key, i, cb) : kv8_v_at(key, i)] = (uint8_t)kv8_codes2(y[k] * inverse, 0.f);
    }
    if (lane == 0) (is_k ? k_exp : v_exp)[place * SX_PAGE + key] = (uint8_t)e;
  }
}

// The same for many tokens at head size 64 or 128, the whole head rotated or nothing.  Blocks of one kind take the q and k heads of four tokens, 64
// threads a token and 16 elements a lane (8 of either half of the head, so that rotation stays within the lane and a key's codes leave as 8-byte
// stores).  Blocks of the other kind take values: a value page lies dim by dim, and a token alone would write a byte here and there (measured in
// all: 338 us for 8,191 tokens of 48 heads of 128, where bytes take 28.6).  There a thread has two dims of up to 16 tokens that share 16
// neighbouring places of a page, finds the rows' largest magnitudes with its warp by 31 exchanges for all 16 tokens, and stores 16 bytes a dim.
// (One kernel: 16 rows of values one behind the other are mostly waiting, 23 us alone.)
// 8,191 tokens of 48 heads of 128 in bfloat16: 43 us, 4.3 TB/s (float32 65 us).  What counts is how many rows are under way: two blocks an SM take 60 us,
// three (gains in registers beside the angles) 48, four 43, five with registers spilled 48; packed arithmetic, two elements an instruction, changes nothing.
template <typename T> struct Kv8Vec;
template <> struct Kv8Vec<bf16> {
  typedef uint4 Raw8;                                            // 8 and 2 elements as they lie in memory
  typedef uint32_t Raw2;
  static __device__ __forceinline__ Raw8 zero8() { return make_uint4(0, 0, 0, 0); }
  static __device__ __forceinline__ Raw2 zero2() { return 0; }
  static __device__ __forceinline__ void floats8(const Raw8& w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ float2 floats2(Raw2 u) { return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)); }
  static __device__ __forceinline__ void store8(bf16* p, const float (&x)[8]) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      u[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <> struct Kv8Vec<float> {
  struct Raw8 { float4 a, b; };
  typedef float2 Raw2;
  static __device__ __forceinline__ Raw8 zero8() { const float4 z = make_float4(0.f, 0.f, 0.f, 0.f); return {z, z}; }
  static __device__ __forceinline__ Raw2 zero2() { return make_float2(0.f, 0.f); }
  static __device__ __forceinline__ void floats8(const Raw8& w, float (&x)[8]) {
    x[0] = w.a.x; x[1] = w.a.y; x[2] = w.a.z; x[3] = w.a.w; x[4] = w.b.x; x[5] = w.b.y; x[6] = w.b.z; x[7] = w.b.w;
  }
  static __device__ __forceinline__ float2 floats2(Raw2 u) { return u; }
  static __device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) reinterpret_cast<float4*>(p)[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
  }
};
__device__ __forceinline__ uint32_t kv8_magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }   // ordered as the magnitudes are, NaN above infinity
__device__ __forceinline__ int kv8_exponent_of(uint32_t top) { return kv8_exponent(__uint_as_float(top), top < 0x7f800000u); }

__device__ __forceinline__ int kv8_page_of(const int* positions, const int* seq_of_token, const int* block_table, int maxp, int n_pages, int t) {
  const int pos = positions[t], page = (unsigned)(pos >> 6) < (unsigned)maxp ? block_table[(size_t)seq_of_token[t] * maxp + (pos >> 6)] : -1;
  return (unsigned)page < (unsigned)n_pages ? page : -1;
}

#define KV8_TOKENS 16
// values of the groups that begin in tokens 16 block .. + 15, of heads first_head, first_head + heads_step, .. (a head is one or two warps)
template <typename T, int HD>
__device__ __forceinline__ void kv8_prepare_v(const T* __restrict__ qkv, uint8_t* __restrict__ v_pages, uint8_t* __restrict__ v_exp,
                                              const int* __restrict__ positions, const int* __restrict__ seq_of_token,
                                              const int* __restrict__ block_table, int maxp, int nh, int nkv, int n_pages, int row, int n_tokens,
                                              int block, int first, int step, uint32_t (*s_top)[KV8_TOKENS]) {
  constexpr int HALF = HD / 2;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // ---- values: the groups of tokens that share 16 places of a page and begin in this block's 16 tokens
  constexpr int WPH = HALF / 32;                                 // warps a head, two dims a lane
  // a group is a run of one sequence's neighbouring positions within 16 places; lane i looks at token t0 + i
  const int t0 = block * KV8_TOKENS, t_ = min(t0 + lane, n_tokens - 1), before = max(t0 - 1, 0);
  const int pos_ = positions[t_], seq_ = seq_of_token[t_];
  int pos_before = __shfl_up_sync(0xffffffffu, pos_, 1), seq_before = __shfl_up_sync(0xffffffffu, seq_, 1);
  if (lane == 0) {
    pos_before = positions[before];
    seq_before = seq_of_token[before];
  }
  const bool starts = t0 + lane == 0 || t0 + lane >= n_tokens || (pos_ & (KV8_TOKENS - 1)) == 0 || seq_ != seq_before || pos_ != pos_before + 1;
  const uint32_t groups = __ballot_sync(0xffffffffu, starts);    // (a bit set where the tokens end, too)
  for (uint32_t left = groups & 0xffffu; left; left &= left - 1) {
    const int i0 = __ffs(left) - 1, t = t0 + i0;
    if (t >= n_tokens) break;
    const uint32_t behind = groups >> i0 >> 1;
    const int n = min(KV8_TOKENS, behind ? __ffs(behind) : KV8_TOKENS), pos = __shfl_sync(0xffffffffu, pos_, i0), key = pos & (SX_PAGE - 1);
    const int page = kv8_page_of(positions, seq_of_token, block_table, maxp, n_pages, t);
    for (int h0 = first * (8 / WPH); h0 < nkv; h0 += step * (8 / WPH)) {
      const int h = h0 + warp / WPH, d = (warp % WPH) * 64 + 2 * lane;
      typename Kv8Vec<T>::Raw2 x[KV8_TOKENS];
      uint32_t top[KV8_TOKENS];
      const T* src = qkv + (size_t)t * row + (size_t)(nh + nkv + h) * HD + d;
#pragma unroll
      for (int i = 0; i < KV8_TOKENS; ++i) x[i] = h < nkv && i < n ? *reinterpret_cast<const typename Kv8Vec<T>::Raw2*>(src + (size_t)i * row) : Kv8Vec<T>::zero2();
#pragma unroll
      for (int i = 0; i < KV8_TOKENS; ++i) {
        const float2 y = Kv8Vec<T>::floats2(x[i]);
        top[i] = max(kv8_magnitude(y.x), kv8_magnitude(y.y));
      }
      // the warp's largest of each token: after the exchanges lane's belongs to token lane >> 1
      int off = 16;
#pragma unroll
      for (int m = KV8_TOKENS; m > 1; m >>= 1, off >>= 1) {
        const bool up = lane & off;
#pragma unroll
        for (int i = 0; i < m / 2; ++i) {
          const uint32_t keep = up ? top[i + m / 2] : top[i], send = up ? top[i] : top[i + m / 2];
          top[i] = max(keep, __shfl_xor_sync(0xffffffffu, send, off));
        }
      }
      top[0] = max(top[0], __shfl_xor_sync(0xffffffffu, top[0], 1));
      if (WPH > 1) {
        __syncthreads();
        if (!(lane & 1)) s_top[warp][lane >> 1] = top[0];
        __syncthreads();
        top[0] = max(s_top[warp & ~(WPH - 1)][lane >> 1], s_top[warp | (WPH - 1)][lane >> 1]);
      }
      const int mine = kv8_exponent_of(top[0]);
      const size_t place = (size_t)max(page, 0) * nkv + min(h, nkv - 1);
      uint32_t lo[4], hi[4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        lo[w] = hi[w] = 0;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const int k = 4 * w + i;
          const float f0 = kv8_inverse(__shfl_sync(0xffffffffu, mine, 2 * k)), f1 = kv8_inverse(__shfl_sync(0xffffffffu, mine, 2 * k + 2));
          const float2 y0 = Kv8Vec<T>::floats2(x[k]), y1 = Kv8Vec<T>::floats2(x[k + 1]);
          lo[w] |= kv8_codes2(y0.x * f0, y1.x * f1) << (8 * i);
          hi[w] |= kv8_codes2(y0.y * f0, y1.y * f1) << (8 * i);
        }
      }
      if (h >= nkv || page < 0) continue;
      uint8_t* dst = v_pages + place * SX_PAGE * HD + kv8_v_at(key, d);
      if (n == KV8_TOKENS) {                                     // (begins at a multiple of 16)
        *reinterpret_cast<uint4*>(dst) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        *reinterpret_cast<uint4*>(dst + SX_PAGE) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      } else {
#pragma unroll
        for (int i = 0; i < KV8_TOKENS; ++i)
          if (i < n) {
            dst[i] = (uint8_t)(lo[i >> 2] >> (8 * (i & 3)));
            dst[SX_PAGE + i] = (uint8_t)(hi[i >> 2] >> (8 * (i & 3)));
          }
      }
      if (warp % WPH == 0 && !(lane & 1) && (lane >> 1) < n) v_exp[place * SX_PAGE + key + (lane >> 1)] = (uint8_t)mine;
    }
  }
}

#define KV8_QK_TOKENS 4
template <typename T, int HD>
__global__ void __launch_bounds__(256, sizeof(T) == 2 ? 4 : 3) kv8_prepare_wide_kernel(
    const T* __restrict__ qkv, T* __restrict__ q_out, uint8_t* __restrict__ k_pages, uint8_t* __restrict__ v_pages, uint8_t* __restrict__ k_exp,
    uint8_t* __restrict__ v_exp, const float* __restrict__ wq, const float* __restrict__ wk, const float* __restrict__ inv_freq, float eps,
    const int* __restrict__ positions, const int* __restrict__ seq_of_token, const int* __restrict__ block_table, int maxp, int nh, int nkv,
    int n_pages, int row, int n_tokens, int v_blocks, int v_shares) {
  constexpr int HALF = HD / 2, LPH = HD / 16, TOK = KV8_QK_TOKENS;       // lanes a head
  __shared__ __align__(16) float s_cs[TOK][HALF], s_sn[TOK][HALF], s_gain[2][HD];
  __shared__ uint32_t s_top[8][KV8_TOKENS];
  pdl_wait();
  pdl_trigger();
  if (blockIdx.x < v_blocks * v_shares) {                        // (first of all: they wait for memory while the others compute)
    kv8_prepare_v<T, HD>(qkv, v_pages, v_exp, positions, seq_of_token, block_table, maxp, nh, nkv, n_pages, row, n_tokens, blockIdx.x / v_shares,
                         blockIdx.x % v_shares, v_shares, s_top);
    return;
  }
  const int lane = threadIdx.x & 31, t0 = (blockIdx.x - v_blocks * v_shares) * TOK, tokens = min(TOK, n_tokens - t0);
  if (inv_freq)
    for (int i = threadIdx.x; i < tokens * HALF; i += 256) {
      const float2 r = kv8_turn(positions[t0 + i / HALF], inv_freq[i % HALF]);
      s_cs[i / HALF][i % HALF] = r.x;
      s_sn[i / HALF][i % HALF] = r.y;
    }
  if (threadIdx.x < 2 * HD) {
    const float* gain = threadIdx.x < HD ? wq : wk;
    if (gain) s_gain[threadIdx.x / HD][threadIdx.x % HD] = gain[threadIdx.x % HD];
  }
  __syncthreads();
  // 64 threads a token: its angles stay in registers over all heads (the gains with them would cost a block an SM)
  constexpr int HPT = 64 / LPH;                                  // heads at a time
  const int tok = threadIdx.x / 64, t = t0 + tok, e0 = (lane % LPH) * 8, h0 = threadIdx.x % 64 / LPH;
  const bool here = tok < tokens;
  const int pos = here ? positions[t] : 0, page = here && k_pages ? kv8_page_of(positions, seq_of_token, block_table, maxp, n_pages, t) : -1;
  float cs[8], sn[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = inv_freq && here ? s_cs[tok][e0 + i] : 1.f;
    sn[i] = inv_freq && here ? s_sn[tok][e0 + i] : 0.f;
  }
#pragma unroll 1
  for (int kind = 0; kind < (k_pages ? 2 : 1); ++kind) {
    const bool gain = kind ? wk != nullptr : wq != nullptr;
    const int n = kind ? nkv : nh;
    typedef typename Kv8Vec<T>::Raw8 Raw;
    const T* src = qkv + (size_t)t * row + (size_t)kind * nh * HD + e0;
    Raw next_a = Kv8Vec<T>::zero8(), next_b = next_a;            // the next head's elements are under way while one is worked at
    if (here && h0 < n) {
      next_a = *reinterpret_cast<const Raw*>(src + (size_t)h0 * HD);
      next_b = *reinterpret_cast<const Raw*>(src + (size_t)h0 * HD + HALF);
    }
#pragma unroll 1
    for (int head = h0; head < (n + HPT - 1) / HPT * HPT; head += HPT) {
      const bool live = here && head < n;
      float a[8], b[8];
      Kv8Vec<T>::floats8(next_a, a);
      Kv8Vec<T>::floats8(next_b, b);
      if (here && head + HPT < n) {
        next_a = *reinterpret_cast<const Raw*>(src + (size_t)(head + HPT) * HD);
        next_b = *reinterpret_cast<const Raw*>(src + (size_t)(head + HPT) * HD + HALF);
      }
      if (gain) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(ss / (float)HD + eps);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 ga = *reinterpret_cast<const float4*>(&s_gain[kind][e0 + i]), gb = *reinterpret_cast<const float4*>(&s_gain[kind][e0 + HALF + i]);
          a[i] = a[i] * inv * ga.x; a[i + 1] = a[i + 1] * inv * ga.y; a[i + 2] = a[i + 2] * inv * ga.z; a[i + 3] = a[i + 3] * inv * ga.w;
          b[i] = b[i] * inv * gb.x; b[i + 1] = b[i + 1] * inv * gb.y; b[i + 2] = b[i + 2] * inv * gb.z; b[i + 3] = b[i + 3] * inv * gb.w;
        }
      }
      if (inv_freq) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = a[i] * cs[i] - b[i] * sn[i], y = a[i] * sn[i] + b[i] * cs[i];
          a[i] = x;
          b[i] = y;
        }
      }
      if (kind == 0) {
        if (!live) continue;
        T* dst = q_out + ((size_t)t * nh + head) * HD + e0;
        Kv8Vec<T>::store8(dst, a);
        Kv8Vec<T>::store8(dst + HALF, b);
        continue;
      }
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, max(kv8_magnitude(a[i]), kv8_magnitude(b[i])));
#pragma unroll
      for (int o = LPH / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      if (!live || page < 0) continue;
      const int e = kv8_exponent_of(top), key = pos & (SX_PAGE - 1);
      const float inverse = kv8_inverse(e);
      const size_t place = (size_t)page * nkv + head;
      uint32_t ca[2], cb[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        ca[i] = kv8_codes2(a[4 * i] * inverse, a[4 * i + 1] * inverse) | kv8_codes2(a[4 * i + 2] * inverse, a[4 * i + 3] * inverse) << 16;
        cb[i] = kv8_codes2(b[4 * i] * inverse, b[4 * i + 1] * inverse) | kv8_codes2(b[4 * i + 2] * inverse, b[4 * i + 3] * inverse) << 16;
      }
      uint8_t* dst = k_pages + place * SX_PAGE * HD;
      *reinterpret_cast<uint2*>(dst + kv8_k_at(key, e0, 64)) = make_uint2(ca[0], ca[1]);
      *reinterpret_cast<uint2*>(dst + kv8_k_at(key, e0 + HALF, 64)) = make_uint2(cb[0], cb[1]);
      if (e0 == 0) k_exp[place * SX_PAGE + key] = (uint8_t)e;
    }
  }
}

// qkv: rows of `row` elements, q heads, k heads and v heads first (q heads alone where k_pages is null and nothing is written).
// wide: by the kernels for many tokens
extern "C" int sx_kv8_prepare(const void* qkv, void* q_out, void* k_pages, void* v_pages, void* k_exp, void* v_exp, const float* wq,
                              const float* wk, const float* inv_freq, int rotary_dim, float eps, const int* positions,
                              const int* seq_of_token, const int* block_table, int maxp, int n_tokens, int nh, int nkv, int hd,
                              int n_pages, int row, int wide, int dt, cudaStream_t stream) {
  if (n_tokens <= 0) return 0;
  if (hd <= 0 || hd % 16 || hd > KV8_MAX_HD || rotary_dim < 0 || rotary_dim > hd || (rotary_dim & 1) || nh < 0 || nkv <= 0)
    return SX_ERR_SIZE;
  const int heads = nh + (k_pages ? 2 * nkv : 0), groups = (heads + KV8_WARPS - 1) / KV8_WARPS;
  if (heads == 0) return 0;
  const size_t es = dt == SX_F32 ? 4 : 2;
  if (wide) {
    if ((hd != 64 && hd != 128) || (inv_freq && rotary_dim != hd)) return SX_ERR_SIZE;
    if (dt != SX_F32 && dt != SX_BF16) return SX_ERR_DTYPE;
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)wq | (uintptr_t)wk | row * es) & 15) return SX_ERR_ALIGN;
    const int v_blocks = v_pages ? (n_tokens + KV8_TOKENS - 1) / KV8_TOKENS : 0, v_shares = (nkv * (hd / 64) + 7) / 8;
    const dim3 blocks(v_blocks * v_shares + (n_tokens + KV8_QK_TOKENS - 1) / KV8_QK_TOKENS);
#define KV8_WIDE(T, HD)                                                                                                                                \
  sx_launch(kv8_prepare_wide_kernel<T, HD>, blocks, dim3(256), 0, stream, (const T*)qkv, (T*)q_out, (uint8_t*)k_pages, (uint8_t*)v_pages,               \
            (uint8_t*)k_exp, (uint8_t*)v_exp, wq, wk, inv_freq, eps, positions, seq_of_token, block_table, maxp, nh, nkv, n_pages, row, n_tokens,        \
            v_blocks, v_shares)
    if (dt == SX_F32) return hd == 64 ? KV8_WIDE(float, 64) : KV8_WIDE(float, 128);
    return hd == 64 ? KV8_WIDE(bf16, 64) : KV8_WIDE(bf16, 128);
  }
  // few tokens: a block for every eight heads; many: a block walks its token's heads and makes the angles once
  const dim3 grid(n_tokens, n_tokens * groups <= 4 * sx_sm_count() ? groups : 1);
  if (dt == SX_F32)
    return sx_launch(kv8_prepare_kernel<float>, grid, dim3(KV8_WARPS * 32), 0, stream, (const float*)qkv, (float*)q_out, (uint8_t*)k_pages,
                     (uint8_t*)v_pages, (uint8_t*)k_exp, (uint8_t*)v_exp, wq, wk, inv_freq, rotary_dim, eps, positions, seq_of_token,
                     block_table, maxp, nh, nkv, hd, n_pages, row);
  if (dt == SX_BF16)
    return sx_launch(kv8_prepare_kernel<bf16>, grid, dim3(KV8_WARPS * 32), 0, stream, (const bf16*)qkv, (bf16*)q_out, (uint8_t*)k_pages,
                     (uint8_t*)v_pages, (uint8_t*)k_exp, (uint8_t*)v_exp, wq, wk, inv_freq, rotary_dim, eps, positions, seq_of_token,
                     block_table, maxp, nh, nkv, hd, n_pages, row);
  return SX_ERR_DTYPE;
}

// ---------------------------------------------------------------------------------------
// Pages read back: page i of the result holds page page_idx[i] of sequence page_seq[i] as [kv heads][64][hd] in T, rows
// behind the sequence's end as zeros.  A block a (page, kv head), bound by its bytes.  A lane of keys takes 8 codes of a
// row at a time (16 bytes of bfloat16); a lane of values takes 8 dims of 4 keys, one word a dim, turns the bytes around in registers and
// stores 16 bytes a key: 8 lanes beside one another read 32 bytes of a dim, 4 write 64 of a key.
// page_from (attention): page i's rows before page_from[i], which no token of the step sees, are zeros, too, and a value row that is not finite comes back as zeros
// and its key row as NaN instead.  Kernels that multiply a page's values with weights of several tokens then give NaN to the tokens that see the
// row, by their scores, and to no others (a weight of zero times NaN would).
// Eight sequences of 4,969 to 12,000 tokens, 8 heads of 128, to bfloat16: 70 to 73 us for 411 MB moved, 5.6 to 5.8 TB/s: HBM, nine tenths of a plain copy's rate.
// ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void kv8_store8(T* dst, const uint32_t (&pairs)[4], float f) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = kv8_float2(pairs[i]);
    x[2 * i] = f != 0.f ? v.x * f : 0.f;
    x[2 * i + 1] = f != 0.f ? v.y * f : 0.f;
  }
  Kv8Vec<T>::store8(dst, x);
}
// HD: the head size where it is 64 or 128 (all loads of a block are then under way at once), 0 for any
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv8_read_kernel(
    const uint8_t* __restrict__ k_pages, const uint8_t* __restrict__ v_pages, const uint8_t* __restrict__ k_exp,
    const uint8_t* __restrict__ v_exp, T* __restrict__ k_out, T* __restrict__ v_out, const int* __restrict__ page_seq,
    const int* __restrict__ page_idx, const int* __restrict__ page_from, const int* __restrict__ seq_lens, const int* __restrict__ block_table,
    int maxp, int nkv, int hd_, int n_pages) {
  __shared__ float s_k[SX_PAGE], s_v[SX_PAGE];
  pdl_wait();
  pdl_trigger();
  const int hd = HD ? HD : hd_, groups = hd / 8, cb = kv8_block(hd);     // groups of 8 dims
  const int i = blockIdx.x, kvh = blockIdx.y;
  const int s = page_seq[i], j = page_idx[i];
  const int page = block_table[(size_t)s * maxp + j];
  const bool ok = page >= 0 && page < n_pages;
  const int held = ok ? min(SX_PAGE, max(0, seq_lens[s] - j * SX_PAGE)) : 0, from_key = page_from ? page_from[i] : 0;
  const size_t from = (size_t)(ok ? page : 0) * nkv + kvh, to = ((size_t)i * nkv + kvh) * SX_PAGE * hd;
  const uint8_t *k = k_pages + from * SX_PAGE * hd, *v = v_pages + from * SX_PAGE * hd;
  constexpr int NK = HD ? HD / 32 : 1, NV = 1;     // items of a thread, where that is known
  // items of values, by bits: 3 of the word of 4 keys, 2 of the group of dims, 1 of the word, the group's rest
  auto v_key = [](int o) { return ((o & 7) | (o >> 2 & 8)) * 4; };
  auto v_group = [](int o) { return (o >> 3 & 3) | (o >> 6) * 4; };
  uint2 kw[NK];
  uint32_t vw[NV][8];
  if (HD) {
#pragma unroll
    for (int n = 0; n < NK; ++n) {
      const int o = threadIdx.x + 256 * n;
      kw[n] = *reinterpret_cast<const uint2*>(k + kv8_k_at(o / groups, o % groups * 8, cb));
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      const int o = threadIdx.x + 256 * n;
      if (o < groups * 16)
#pragma unroll
        for (int d = 0; d < 8; ++d) vw[n][d] = *reinterpret_cast<const uint32_t*>(v + kv8_v_at(v_key(o), v_group(o) * 8 + d));
    }
  }
  if (threadIdx.x < 2 * SX_PAGE) {
    const int key = threadIdx.x & (SX_PAGE - 1), ve = v_exp[from * SX_PAGE + key];
    const bool there = key < held && key >= from_key, gone = page_from && ve == KV8_NAN;      // (a factor of zero: zeros, whatever the codes are)
    if (threadIdx.x < SX_PAGE) s_k[key] = there ? kv8_scale(gone ? KV8_NAN : k_exp[from * SX_PAGE + key]) : 0.f;
    else s_v[key] = there && !gone ? kv8_scale(ve) : 0.f;
  }
  __syncthreads();
  auto put_k = [&](int o, const uint2 w) {
    const int key = o / groups, d = o % groups * 8;
    const uint32_t pairs[4] = {w.x, w.x >> 16, w.y, w.y >> 16};
    kv8_store8<T>(k_out + to + key * hd + d, pairs, s_k[key]);
  };
  auto put_v = [&](int o, const uint32_t (&w)[8]) {
    const int key = v_key(o), group = v_group(o);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      uint32_t pairs[4];
#pragma unroll
      for (int d = 0; d < 4; ++d) pairs[d] = __byte_perm(w[2 * d], w[2 * d + 1], n | (4 + n) << 4);
      kv8_store8<T>(v_out + to + (key + n) * hd + group * 8, pairs, s_v[key + n]);
    }
  };
  if constexpr (HD != 0) {
#pragma unroll
    for (int n = 0; n < NK; ++n) put_k(threadIdx.x + 256 * n, kw[n]);
#pragma unroll
    for (int n = 0; n < NV; ++n)
      if (threadIdx.x + 256 * n < groups * 16) put_v(threadIdx.x + 256 * n, vw[n]);
  } else {
    for (int o = threadIdx.x; o < SX_PAGE * groups; o += 256) put_k(o, *reinterpret_cast<const uint2*>(k + kv8_k_at(o / groups, o % groups * 8, cb)));
    for (int o = threadIdx.x; o < (groups + 3) / 4 * 64; o += 256) {
      if (v_group(o) >= groups) continue;
      uint32_t w[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) w[d] = *reinterpret_cast<const uint32_t*>(v + kv8_v_at(v_key(o), v_group(o) * 8 + d));
      put_v(o, w);
    }
  }
}

extern "C" int sx_kv8_read(const void* k_pages, const void* v_pages, const void* k_exp, const void* v_exp, void* k_out, void* v_out,
                           const int* page_seq, const int* page_idx, const int* page_from, int n_out, const int* seq_lens,
                           const int* block_table, int maxp, int nkv, int hd, int n_pages, int dt, cudaStream_t stream) {
  if (n_out <= 0) return 0;
  if (hd <= 0 || hd % 16 || hd > KV8_MAX_HD || nkv <= 0 || nkv > 65535) return SX_ERR_SIZE;
  if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15) return SX_ERR_ALIGN;
  const dim3 grid(n_out, nkv);
#define KV8_READ(T, HD)                                                                                                                            \
  sx_launch(kv8_read_kernel<T, HD>, grid, dim3(256), 0, stream, (const uint8_t*)k_pages, (const uint8_t*)v_pages, (const uint8_t*)k_exp,             \
            (const uint8_t*)v_exp, (T*)k_out, (T*)v_out, page_seq, page_idx, page_from, seq_lens, block_table, maxp, nkv, hd, n_pages)
  if (dt == SX_F32) return hd == 64 ? KV8_READ(float, 64) : hd == 128 ? KV8_READ(float, 128) : KV8_READ(float, 0);
  if (dt == SX_BF16) return hd == 64 ? KV8_READ(bf16, 64) : hd == 128 ? KV8_READ(bf16, 128) : KV8_READ(bf16, 0);
  return SX_ERR_DTYPE;
}

// ---------------------------------------------------------------------------------------
// Attention of single tokens over the pages: every head size, type and option.
//
// A block serves up to four query heads of a kv head (a group of more takes several blocks) over a share of the sequence's
// visible pages; its warps take the share's pages in turn, each with a softmax of its own (running maximum and sum), joined in
// shared memory at the end.  In a page a lane has two keys in the scores (a key's codes are 16-byte loads, queries come from
// shared memory and serve all lanes) and hd / 32 dims in p v (a dim's 64 keys are four loads).  All sums in 32 bits by FFMA.
// ---------------------------------------------------------------------------------------
#define KV8_HEADS 4
struct Kv8Rows {
  const uint8_t *k, *v, *ke, *ve;
  const int *seq_lens, *block_table;
  const float* sinks;
  float *part_o, *part_ml;
  int maxp, n_pages, nh, nkv, hd, window, chunk, n_splits, out_stride;
  float scale, softcap, out_scale;
};

template <typename T, int NI>
__global__ void __launch_bounds__(KV8_WARPS * 32) kv8_rows_kernel(const T* __restrict__ q, T* __restrict__ out, const Kv8Rows a) {
  extern __shared__ float4 smem4[];
  float* q_s = reinterpret_cast<float*>(smem4);                              // [KV8_HEADS][hd]
  const int hd = a.hd, G = a.nh / a.nkv, per_kv = (G + KV8_HEADS - 1) / KV8_HEADS;
  float* p_s = q_s + KV8_HEADS * hd;                                         // [KV8_WARPS][KV8_HEADS][64]
  float* o_s = p_s + KV8_WARPS * KV8_HEADS * SX_PAGE;                        // [KV8_WARPS][KV8_HEADS][hd]
  __shared__ float s_m[KV8_WARPS][KV8_HEADS], s_l[KV8_WARPS][KV8_HEADS], s_r[KV8_HEADS];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.x, kvh = blockIdx.y / per_kv, g0 = (blockIdx.y % per_kv) * KV8_HEADS, seq = blockIdx.z;
  const int gn = min(KV8_HEADS, G - g0), h0 = kvh * G + g0;
  const int len = a.seq_lens[seq], pos = len - 1;
  int lo = a.window > 0 ? max(0, len - a.window) : 0;
  if (a.chunk > 0 && pos >= 0) lo = max(lo, pos / a.chunk * a.chunk);
  const int p_first = lo >> 6, p_end = min((len + 63) >> 6, a.maxp);
  const int per = (max(0, p_end - p_first) + a.n_splits - 1) / a.n_splits;
  const int p0 = p_first + split * per, p1 = min(p_end, p0 + per);
  // queries, each row scaled by a power of two to a largest magnitude of 1 to 2, so that no sum of products with codes leaves the range
  for (int g = warp; g < KV8_HEADS; g += KV8_WARPS) {
    const T* src = q + ((size_t)seq * a.nh + h0 + g) * hd;
    float top = 0.f;
    bool finite = true;
    for (int i = lane; g < gn && i < hd; i += 32) {
      const float x = to_f32(src[i]);
      top = fmaxf(top, fabsf(x));
      finite = finite && fabsf(x) < INFINITY;
    }
    finite = __all_sync(0xffffffffu, finite);
    const int x = min(max(__float_as_int(warp_max(top)) >> 23, 1), 253);
    const float down = __int_as_float((254 - x) << 23);
    for (int i = lane; i < hd; i += 32) q_s[g * hd + i] = g < gn ? to_f32(src[i]) * down : 0.f;
    if (lane == 0) s_r[g] = finite ? __int_as_float(x << 23) * a.scale : __int_as_float(0x7fffffff);
  }
  __syncthreads();
  const int cb = kv8_block(hd);
  float m[KV8_HEADS], l[KV8_HEADS], o[KV8_HEADS][NI];
#pragma unroll
  for (int g = 0; g < KV8_HEADS; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < NI; ++i) o[g][i] = 0.f;
  }
  float* pw = p_s + warp * KV8_HEADS * SX_PAGE;
  for (int p = p0 + warp; p < p1; p += KV8_WARPS) {
    const int page = a.block_table[(size_t)seq * a.maxp + p];
    if (page < 0 || page >= a.n_pages) continue;
    const size_t place = (size_t)page * a.nkv + kvh;
    const uint8_t* kp = a.k + place * SX_PAGE * hd;
    const uint8_t* vp = a.v + place * SX_PAGE * hd;
    const int v0 = max(0, lo - p * SX_PAGE), v1 = min(SX_PAGE, len - p * SX_PAGE);     // visible keys of the page
    float s[2][KV8_HEADS];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int key = lane + 32 * h;
#pragma unroll
      for (int g = 0; g < KV8_HEADS; ++g) s[h][g] = 0.f;
      for (int d = 0; d < hd; d += 16) {
        float x[16];
        kv8_float16(*reinterpret_cast<const uint4*>(kp + kv8_k_at(key, d, cb)), x);
#pragma unroll
        for (int g = 0; g < KV8_HEADS; ++g) {
          float part = 0.f;                                          // (sums of 16, then of those: fewer roundings of large sums)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 y = *reinterpret_cast<const float4*>(q_s + g * hd + d + 4 * i);
            part = fmaf(y.x, x[4 * i], fmaf(y.y, x[4 * i + 1], fmaf(y.z, x[4 * i + 2], fmaf(y.w, x[4 * i + 3], part))));
          }
          s[h][g] += part;
        }
      }
    }
    const float kf[2] = {kv8_scale(a.ke[place * SX_PAGE + lane]), kv8_scale(a.ke[place * SX_PAGE + lane + 32])};
    const float vf[2] = {kv8_scale(a.ve[place * SX_PAGE + lane]), kv8_scale(a.ve[place * SX_PAGE + lane + 32])};
    __syncwarp();
#pragma unroll
    for (int g = 0; g < KV8_HEADS; ++g) {
      float top = m[g];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = lane + 32 * h;
        float z = s[h][g] * (kf[h] * s_r[g]);                        // (up to 2^18 times a power of up to 2^119: the powers go together first)
        if (a.softcap > 0.f) z = a.softcap * tanhf(z / a.softcap);
        s[h][g] = key >= v0 && key < v1 ? z : -INFINITY;
        top = fmaxf(top, s[h][g]);
      }
      top = warp_max(top);
      const float base = top == -INFINITY ? 0.f : top, shrink = expf(m[g] - base);
      m[g] = top;
      float sum = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = lane + 32 * h;
        const float w = expf(s[h][g] - base);
        sum += w;
        pw[g * SX_PAGE + key] = key >= v0 && key < v1 ? w * vf[h] : 0.f;
      }
      l[g] = l[g] * shrink + warp_sum(sum);
#pragma unroll
      for (int i = 0; i < NI; ++i) o[g][i] *= shrink;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int d = lane + 32 * i;
      if (d >= hd) continue;
#pragma unroll
      for (int c = 0; c < SX_PAGE; c += 16) {
        float x[16];
        kv8_float16(*reinterpret_cast<const uint4*>(vp + kv8_v_at(c, d)), x);
        if (c < v0 || c + 16 > v1) {                                 // codes of keys that are not seen may be anything
#pragma unroll
          for (int n = 0; n < 16; ++n)
            if (c + n < v0 || c + n >= v1) x[n] = 0.f;
        }
#pragma unroll
        for (int g = 0; g < KV8_HEADS; ++g) {
          float part = 0.f;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float4 w = *reinterpret_cast<const float4*>(pw + g * SX_PAGE + c + 4 * n);
            part = fmaf(w.x, x[4 * n], fmaf(w.y, x[4 * n + 1], fmaf(w.z, x[4 * n + 2], fmaf(w.w, x[4 * n + 3], part))));
          }
          o[g][i] += part;
        }
      }
    }
  }
#pragma unroll
  for (int g = 0; g < KV8_HEADS; ++g) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
      if (lane + 32 * i < hd) o_s[(warp * KV8_HEADS + g) * hd + lane + 32 * i] = o[g][i];
    if (lane == 0) {
      s_m[warp][g] = m[g];
      s_l[warp][g] = l[g];
    }
  }
  __syncthreads();
  for (int n = threadIdx.x; n < gn * hd; n += KV8_WARPS * 32) {
    const int g = n / hd, d = n % hd, head = h0 + g;
    float M = -INFINITY;
    for (int w = 0; w < KV8_WARPS; ++w) M = fmaxf(M, s_m[w][g]);
    const bool last = a.n_splits == 1;
    const bool sink = last && a.sinks;
    if (sink) M = fmaxf(M, a.sinks[head]);
    const float base = M == -INFINITY ? 0.f : M;
    float L = sink ? expf(a.sinks[head] - base) : 0.f, O = 0.f;
    for (int w = 0; w < KV8_WARPS; ++w) {
      const float f = expf(s_m[w][g] - base);
      L += s_l[w][g] * f;
      O += o_s[(w * KV8_HEADS + g) * hd + d] * f;
    }
    const size_t r = (size_t)seq * a.nh + head;
    if (last) {
      out[(size_t)seq * a.out_stride + head * hd + d] = from_f32<T>(L == 0.f ? 0.f : O / L * a.out_scale);
    } else {
      a.part_o[(r * a.n_splits + split) * hd + d] = O;
      if (d == 0) reinterpret_cast<float2*>(a.part_ml)[r * a.n_splits + split] = make_float2(M, L);
    }
  }
}

// the shares of a row joined: a block a (sequence, head), a thread a dim
template <typename T>
__global__ void kv8_rows_merge_kernel(T* __restrict__ out, const Kv8Rows a) {
  pdl_wait();
  pdl_trigger();
  const int seq = blockIdx.x / a.nh, head = blockIdx.x % a.nh, d = threadIdx.x;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)blockIdx.x * a.n_splits;
  const float* po = a.part_o + (size_t)blockIdx.x * a.n_splits * a.hd + d;
  float M = a.sinks ? a.sinks[head] : -INFINITY;
  for (int i = 0; i < a.n_splits; ++i) M = fmaxf(M, ml[i].x);
  const float base = M == -INFINITY ? 0.f : M;
  float L = a.sinks ? expf(a.sinks[head] - base) : 0.f, O = 0.f;
  for (int i = 0; i < a.n_splits; ++i) {
    const float f = expf(ml[i].x - base);
    L += ml[i].y * f;
    O += po[(size_t)i * a.hd] * f;
  }
  out[(size_t)seq * a.out_stride + head * a.hd + d] = from_f32<T>(L == 0.f ? 0.f : O / L * a.out_scale);
}

template <typename T>
static int kv8_rows_launch(const void* q, void* out, int S, const Kv8Rows& a, cudaStream_t stream) {
  const int G = a.nh / a.nkv, per_kv = (G + KV8_HEADS - 1) / KV8_HEADS;
  const dim3 grid(a.n_splits, a.nkv * per_kv, S), block(KV8_WARPS * 32);
  const size_t smem = (size_t)(KV8_HEADS * a.hd + KV8_WARPS * KV8_HEADS * (SX_PAGE + a.hd)) * sizeof(float);
  int rc;
  if (a.hd <= 32) rc = sx_launch(kv8_rows_kernel<T, 1>, grid, block, smem, stream, (const T*)q, (T*)out, a);
  else if (a.hd <= 64) rc = sx_launch(kv8_rows_kernel<T, 2>, grid, block, smem, stream, (const T*)q, (T*)out, a);
  else if (a.hd <= 128) rc = sx_launch(kv8_rows_kernel<T, 4>, grid, block, smem, stream, (const T*)q, (T*)out, a);
  else rc = sx_launch(kv8_rows_kernel<T, 8>, grid, block, smem, stream, (const T*)q, (T*)out, a);
  if (rc || a.n_splits == 1) return rc;
  return sx_launch(kv8_rows_merge_kernel<T>, dim3(S * a.nh), dim3(a.hd), 0, stream, (T*)out, a);
}

extern "C" int sx_kv8_rows(const void* q, void* out, const void* k, const void* v, const void* k_exp, const void* v_exp, const int* seq_lens,
                           const int* block_table, int maxp, int S, int nh, int nkv, int hd, int n_pages, float scale, int window,
                           float softcap, const float* sinks, int chunk, int out_stride, float out_scale, int n_splits, float* part_o,
                           float* part_ml, int dt, cudaStream_t stream) {
  if (S <= 0) return 0;
  if (hd <= 0 || hd % 16 || hd > KV8_MAX_HD || nkv <= 0 || nh <= 0 || nh % nkv || n_splits < 1 || S > 65535 ||
      (long long)nkv * ((nh / nkv + KV8_HEADS - 1) / KV8_HEADS) > 65535 || (n_splits > 1 && (!part_o || !part_ml)))
    return SX_ERR_SIZE;
  if (((uintptr_t)k | (uintptr_t)v) & 15) return SX_ERR_ALIGN;
  const Kv8Rows a = {(const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_exp, (const uint8_t*)v_exp, seq_lens, block_table, sinks, part_o,
                     part_ml, maxp, n_pages, nh, nkv, hd, window, chunk, n_splits, out_stride, scale, softcap, out_scale};
  if (dt == SX_F32) return kv8_rows_launch<float>(q, out, S, a, stream);
  if (dt == SX_BF16) return kv8_rows_launch<bf16>(q, out, S, a, stream);
  return SX_ERR_DTYPE;
}
