// Attention of portions over a cache in eight bits (kv8.cuh), on the codes themselves: bfloat16 and float32 queries, head size 64 or 128, up to 64
// query heads a kv head.
//
// Rows of a tile are the query heads of one kv head of some tokens of one sequence, 64 of them, so that a page's codes serve them all; a warp
// has 16 and walks the tile's pages with a running maximum and sum of its rows.  Both products are matrix instructions on 16 rows x 8 keys (or dims):
//   * q k^T in bfloat16: m16n8k32 on the codes as they are, a query as the sum of two e4m3 numbers (as single tokens have it: elements down to 2^-9 of a
//     power just below the row's largest are exact, smaller ones off by at most 2^-18 of it).  In float32: m16n8k16 in half precision, which e4m3 becomes
//     exactly, a query as the sum of two halves: 22 bits of an element, down to 2^-39 of the row's largest.  (float32 sums in the tensor cores drop what
//     a 32-bit addition would round: chains are of four and eight instructions, their results are added by plain additions.)
//   * p v: m16n8k16, values as exact halves.  A thread's scores are keys 16 t + 2 j + {0, 1}, which are the weights its fragments want, and a row of codes
//     of one dim is one 16-byte load: nothing moves between lanes.  In float32 weights are two halves as well.
//   * Powers of two.  With x the score (base 2) and E a value's exponent, p = 2^(x - m) goes into the denominator, and p 2^E 2^(15 + m - M) into the half
//     precision beside the codes.  m is the running maximum of x and M that of x + E, each rounded UP to an integer: changing either multiplies by exact powers of two,
//     and one exponential serves both.  Weights down to 2^-29 of the row's largest keep 11 bits (22 in float32);
//     down to 2^-24 where all values that a row sees have the format's lowest powers.
// A value that is not finite (exponent 255) has its codes replaced by zeros before the products, and rows that see its key become NaN by their scores: rows
// that do not see it keep their values.  So have values of keys that no token of the tile sees, before its window or chunk and behind its last
// token: what lies there may be anything, a code that is NaN beside any exponent.
//
// Few tiles are cut: a block takes a share of its tile's pages, and a second kernel joins the shares.
//
// Measured (32 heads over 8 of 128): float32, a prompt of 1,500 160 us, 1,500 tokens behind 6,000 1.11 ms; that is 300 TFLOP/s of half-precision products, two
// for each of the formula's, where this instruction's rate is 560: what bounds it is the warps' own work between the products (two blocks an SM by their
// registers).  The same through pages read back and FFMA products takes 638 us and 5.2 ms.  bfloat16, 16 tokens over 20,000 keys: 48 us (read back 91); three
// blocks an SM, with registers spilled for it, 53.
#include "kv8.cuh"

#define KT_ROWS 64               // of a tile: 16 a warp
#define KT_WARPS 4
#define KT_STAGES 3
#define KT_LOG2E 1.44269504f
#define KT_DOWN 3.0517578125e-5f // 2^-15

struct KtArgs {
  const void* q;
  void* out;
  const uint8_t *k, *v, *ke, *ve;
  const int *cu, *past, *block_table;
  const float* sinks;
  float *part_o, *part_ml;       // of cut tiles: [token][head][share][HD] and maximum, sum of each
  int maxp, n_pages, nh, nkv, window, chunk, out_stride, n_tiles, n_splits;
  float scale, softcap, out_scale;
};

__device__ __forceinline__ float kt_pow2(float k) { return __int_as_float(((int)fminf(fmaxf(k, -127.f), 127.f) + 127) << 23); }   // of an integer
__device__ __forceinline__ int kt_lo(const KtArgs& a, int pos) {                     // the first key that position `pos` sees
  int lo = a.window > 0 ? max(0, pos - a.window + 1) : 0;
  return a.chunk > 0 ? max(lo, pos / a.chunk * a.chunk) : lo;
}

template <typename T, int HD>
__global__ void __launch_bounds__(KT_WARPS * 32, 2) kv8_tile_kernel(const KtArgs a) {
  constexpr bool F32 = sizeof(T) == 4;
  constexpr int TILE = SX_PAGE * HD, STAGE = 2 * TILE + 2 * SX_PAGE;
  extern __shared__ __align__(128) unsigned char smem[];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int seq = blockIdx.z, kvh = blockIdx.y, split = blockIdx.x % a.n_splits, tile = a.n_tiles - 1 - blockIdx.x / a.n_splits;     // (long ones first)
  const int G = a.nh / a.nkv, tokens = KT_ROWS / G, t0 = a.cu[seq], n_new = a.cu[seq + 1] - t0, q0 = tile * tokens;
  if (q0 >= n_new) return;
  const int n_tok = min(tokens, n_new - q0), first = a.past[seq] + q0, end = first + n_tok;     // positions of the tile: first .. end - 1
  const int begin = kt_lo(a, first), page0 = begin >> 6, n_pages = max(0, min((end + 63) >> 6, a.maxp) - page0);       // (no token of the tile sees a key before)
  const int per = (n_pages + a.n_splits - 1) / a.n_splits, p0 = page0 + min(split * per, n_pages), p1 = min(p0 + per, page0 + n_pages);
  // the rows of the thread (g, g + 8 of the warp's) and the keys they see
  int tok[2], head[2], lo[2], hi[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = 16 * warp + g + 8 * r;
    tok[r] = row / G;
    head[r] = kvh * G + row - tok[r] * G;
    lo[r] = kt_lo(a, first + tok[r]);
    hi[r] = tok[r] < n_tok ? first + tok[r] + 1 : 0;
  }
  const int tok_a = 16 * warp / G, tok_b = min((16 * warp + 15) / G, n_tok - 1);     // the warp's tokens
  const int some_lo = kt_lo(a, first + tok_a), some_hi = tok_a < n_tok ? first + tok_b + 1 : 0;        // keys that some row of the warp sees,
  const int all_lo = kt_lo(a, first + tok_b), all_hi = first + tok_a + 1;                              // that all do

  const uint32_t smem_a = (uint32_t)__cvta_generic_to_shared(smem);
  auto load = [&](int p) {
    if (p < p1) {
      int page = a.block_table[(size_t)seq * a.maxp + p];
      if ((unsigned)page >= (unsigned)a.n_pages) page = 0;
      const size_t place = (size_t)page * a.nkv + kvh;
      const uint32_t dst = smem_a + (p - p0) % KT_STAGES * STAGE;
      const uint8_t *k = a.k + place * TILE, *v = a.v + place * TILE;
#pragma unroll
      for (int i = 0; i < TILE / (KT_WARPS * 512); ++i) {
        const int at = (i * KT_WARPS * 32 + threadIdx.x) * 16;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst + at), "l"(k + at) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst + TILE + at), "l"(v + at) : "memory");
      }
      if (threadIdx.x < 8) {
        const uint8_t* e = (threadIdx.x < 4 ? a.ke : a.ve) + place * SX_PAGE + 16 * t;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 16;\n" ::"r"(dst + 2 * TILE + 16 * threadIdx.x), "l"(e) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;\n" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < KT_STAGES - 1; ++i) load(p0 + i);

  // queries as two parts, scaled by a power of two
  uint32_t qf[HD / 16][2][F32 ? 4 : 2];     // float32: [steps of 16 dims][part][fragment]; bfloat16: [4 dims][part][row]
  float c[2], m[2], l[2], M[2], o[HD / 8][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const bool on = hi[r] > 0;
    const size_t at = ((size_t)(t0 + q0 + (on ? tok[r] : 0)) * a.nh + head[r]) * HD + 16 * t;
    float x[HD / 4];                        // dims 64 b + 16 t .. + 15
    if constexpr (F32) {
      const float4* src = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.q) + at);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        const float4 y = on ? src[(i >> 2) * 16 + (i & 3)] : make_float4(0.f, 0.f, 0.f, 0.f);
        x[4 * i] = y.x; x[4 * i + 1] = y.y; x[4 * i + 2] = y.z; x[4 * i + 3] = y.w;
      }
    } else {
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const bf16*>(a.q) + at);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const uint4 y = on ? src[(i >> 1) * 8 + (i & 1)] : make_uint4(0, 0, 0, 0);
        const uint32_t u[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
          x[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
      }
    }
    uint32_t top = 0;                       // the largest magnitude by its bits
#pragma unroll
    for (int i = 0; i < HD / 4; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // largest scaled to 2^UP .. 2^(UP + 1)
    constexpr int UP = F32 ? 14 : 7;
    const int e = max((int)(top >> 23), 28);
    const float down = __int_as_float((254 + UP - e) << 23);
    c[r] = (top >= 0x7f800000u ? __int_as_float(0x7fffffff) : __int_as_float((e - UP) << 23)) * a.scale * (a.softcap > 0.f ? 1.f : KT_LOG2E);
#pragma unroll
    for (int k = 0; k < HD / 16; ++k) {
      const float y[4] = {x[4 * k] * down, x[4 * k + 1] * down, x[4 * k + 2] * down, x[4 * k + 3] * down};
      if constexpr (F32) {
        const __half2 h0 = __floats2half2_rn(y[0], y[1]), h1 = __floats2half2_rn(y[2], y[3]);
        const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
        qf[k][0][r] = *reinterpret_cast<const uint32_t*>(&h0);
        qf[k][0][2 + r] = *reinterpret_cast<const uint32_t*>(&h1);
        qf[k][1][r] = kv8_pack2(y[0] - f0.x, y[1] - f0.y);
        qf[k][1][2 + r] = kv8_pack2(y[2] - f1.x, y[3] - f1.y);
      } else {
        const uint32_t c0 = kv8_codes2(y[0], y[1]), c1 = kv8_codes2(y[2], y[3]);
        const float2 f0 = kv8_float2(c0), f1 = kv8_float2(c1);
        qf[k][0][r] = c0 | c1 << 16;
        qf[k][1][r] = kv8_codes2(y[0] - f0.x, y[1] - f0.y) | kv8_codes2(y[2] - f1.x, y[3] - f1.y) << 16;
      }
    }
    m[r] = M[r] = -INFINITY;
    l[r] = 0.f;
  }
#pragma unroll
  for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;

  for (int p = p0; p < p1; ++p) {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(KT_STAGES - 2) : "memory");
    __syncthreads();                        // this page is there, and nobody reads the one before any more
    load(p + KT_STAGES - 1);
    unsigned char* ks = smem + (p - p0) % KT_STAGES * STAGE;
    unsigned char* vs = ks + TILE;
    const int key0 = p * SX_PAGE;
    const uint4 ve4 = *reinterpret_cast<const uint4*>(vs + TILE + SX_PAGE + 16 * t);       // of the thread's keys 16 t ..
    uint32_t ve[4] = {ve4.x, ve4.y, ve4.z, ve4.w};
    uint32_t nan[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) nan[i] = __vcmpeq4(ve[i], 0xffffffffu);
    const bool mend = __any_sync(0xffffffffu, (nan[0] | nan[1] | nan[2] | nan[3]) != 0) || key0 + SX_PAGE > end || key0 < begin;     // (the same in every warp)
    if (mend) {
      uint32_t keep[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 16 * t + 4 * i, n = min(max(end - key, 0), 4), m = min(max(begin - key, 0), 4);      // of these four: m <= i < n are keys that somebody of the tile may see
        keep[i] = (n == 4 ? ~0u : (1u << (8 * n)) - 1u) & (m == 4 ? 0u : ~0u << (8 * m)) & ~nan[i];
        ve[i] &= ~nan[i];
      }
      for (int at = threadIdx.x * 16; at < TILE; at += KT_WARPS * 512) {            // (a thread's chunks are all of its 16 keys)
        uint4 w = *reinterpret_cast<uint4*>(vs + at);
        w.x &= keep[0]; w.y &= keep[1]; w.z &= keep[2]; w.w &= keep[3];
        *reinterpret_cast<uint4*>(vs + at) = w;
      }
      __syncthreads();
    }
    if (key0 >= some_hi || key0 + SX_PAGE <= some_lo) continue;          // nothing for this warp
    // ---- scores
    float s[8][4];                          // keys 16 t + 2 j + {0, 1}, rows g and g + 8
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned char* row = ks + (16 * (g >> 1) + 2 * j + (g & 1)) * 64 + 16 * t;
      float acc[HD / 64][4], rest[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int b = 0; b < HD / 64; ++b) {
        acc[b][0] = acc[b][1] = acc[b][2] = acc[b][3] = 0.f;
        const uint4 w4 = *reinterpret_cast<const uint4*>(row + b * 4096);
        const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
        if constexpr (F32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = 4 * b + i;
            uint32_t b0, b1;
            kv8_half4(w[i], b0, b1);
            kv8_mma_f16(acc[b], qf[k][0][0], qf[k][0][1], qf[k][0][2], qf[k][0][3], b0, b1);
            kv8_mma_f16(rest, qf[k][1][0], qf[k][1][1], qf[k][1][2], qf[k][1][3], b0, b1);
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int k = 4 * b + 2 * h;
            kv8_mma_e4m3(acc[b], qf[k][0][0], qf[k][0][1], qf[k + 1][0][0], qf[k + 1][0][1], w[2 * h], w[2 * h + 1]);
            kv8_mma_e4m3(rest, qf[k][1][0], qf[k][1][1], qf[k + 1][1][0], qf[k + 1][1][1], w[2 * h], w[2 * h + 1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) s[j][i] = (HD == 128 ? acc[0][i] + acc[HD / 64 - 1][i] : acc[0][i]) + rest[i];
    }
    const uint4 ke4 = *reinterpret_cast<const uint4*>(vs + TILE + 16 * t);
    const uint32_t ke[4] = {ke4.x, ke4.y, ke4.z, ke4.w};
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = 2 * (j & 1) + e;     // 2^(e - 127) from the byte's bits (255: an infinity, which times the NaN of such a row's codes is NaN)
        const float kf = __uint_as_float((at < 3 ? ke[j >> 1] << (23 - 8 * at) : ke[j >> 1] >> 1) & 0x7f800000u);
#pragma unroll
        for (int r = 0; r < 2; ++r) s[j][2 * r + e] *= kf * c[r];
      }
    if (a.softcap > 0.f) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[j][i] = a.softcap * KT_LOG2E * tanhf(s[j][i] / a.softcap);
    }
    if (mend || key0 < all_lo || key0 + SX_PAGE > all_hi) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = key0 + 16 * t + 2 * j + e;
          const bool bad = nan[j >> 1] >> (16 * (j & 1) + 8 * e) & 1;
#pragma unroll
          for (int r = 0; r < 2; ++r) s[j][2 * r + e] = key < lo[r] || key >= hi[r] ? -INFINITY : bad ? __int_as_float(0x7fffffff) : s[j][2 * r + e];
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[i >> 1] = fmaxf(top[i >> 1], s[j][i]);
    float most[2] = {0.f, 0.f}, base[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      top[r] = ceilf(top[r]);
      base[r] = top[r] == -INFINITY ? 0.f : top[r];
      l[r] *= m[r] == top[r] ? 1.f : kt_pow2(m[r] - top[r]);
      m[r] = top[r];
    }
    // ---- weights
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int at = 2 * (j & 1) + e;
        const float vf = __uint_as_float((at < 3 ? ve[j >> 1] << (23 - 8 * at) : ve[j >> 1] >> 1) & 0x7f800000u);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float w = kv8_ex2(s[j][2 * r + e] - base[r]);
          l[r] += w;
          s[j][2 * r + e] = w * vf;
          most[r] = fmaxf(most[r], s[j][2 * r + e]);
        }
      }
    float up[2], shrink[2];
    bool moved = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 1));
      most[r] = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], 2));
      // (M stays within 112 of m: 2^(15 + m - M) is then a float32 number, and weights are no smaller for values whose powers are all below 2^-112)
      const float next = fmaxf(M[r], m[r] + (float)max((__float_as_int(most[r]) >> 23) - 126, -112));
      shrink[r] = M[r] == next ? 1.f : kt_pow2(M[r] - next);
      moved = moved || M[r] != next;
      M[r] = next;
      up[r] = m[r] == -INFINITY ? 1.f : kt_pow2(15.f + m[r] - next);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int d = 0; d < HD / 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] *= shrink[i >> 1];
    }
    uint32_t w0[8][2], w1[F32 ? 8 : 1][2];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float x = s[j][2 * r] * up[r], y = s[j][2 * r + 1] * up[r];
        w0[j][r] = kv8_pack2(x, y);
        if constexpr (F32) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w0[j][r]));
          w1[j][r] = kv8_pack2(x - f.x, y - f.y);
        }
      }
    // ---- p v
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      const uint4 u4 = *reinterpret_cast<const uint4*>(vs + (8 * d + g) * 64 + 16 * t);
      const uint32_t u[4] = {u4.x, u4.y, u4.z, u4.w};
      if constexpr (F32) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f}, rest[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t b0, b1;
          kv8_half4(u[k], b0, b1);
          kv8_mma_f16(acc, w0[2 * k][0], w0[2 * k][1], w0[2 * k + 1][0], w0[2 * k + 1][1], b0, b1);
          kv8_mma_f16(rest, w1[2 * k][0], w1[2 * k][1], w1[2 * k + 1][0], w1[2 * k + 1][1], b0, b1);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) o[d][i] += acc[i] + rest[i];
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t b0, b1;
          kv8_half4(u[k], b0, b1);
          kv8_mma_f16(o[d], w0[2 * k][0], w0[2 * k][1], w0[2 * k + 1][0], w0[2 * k + 1][1], b0, b1);
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;\n" ::: "memory");
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float sum = l[r];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    if (hi[r] == 0) continue;
    // 2^-15 o is 2^-M times sum 2^(x + E) code; times 2^(M - m) it is the sum of p 2^E code
    float f = m[r] == -INFINITY ? 0.f : kt_pow2(M[r] - m[r]);
    const size_t row = (size_t)(t0 + q0 + tok[r]) * a.nh + head[r];
    if (a.n_splits > 1) {
      float* dst = a.part_o + (row * a.n_splits + split) * HD + 2 * t;
#pragma unroll
      for (int d = 0; d < HD / 8; ++d) *reinterpret_cast<float2*>(dst + 8 * d) = make_float2(o[d][2 * r] * KT_DOWN * f, o[d][2 * r + 1] * KT_DOWN * f);
      if (t == 0) reinterpret_cast<float2*>(a.part_ml)[row * a.n_splits + split] = make_float2(m[r], sum);
      continue;
    }
    if (a.sinks) {
      const float sink = a.sinks[head[r]] * KT_LOG2E, all = fmaxf(m[r], sink), b = all == -INFINITY ? 0.f : all, less = kv8_ex2(m[r] - b);
      sum = sum * less + kv8_ex2(sink - b);
      f *= less;
    }
    f = sum == 0.f ? 0.f : f / sum * a.out_scale;
    T* dst = reinterpret_cast<T*>(a.out) + (size_t)(t0 + q0 + tok[r]) * a.out_stride + head[r] * HD + 2 * t;
#pragma unroll
    for (int d = 0; d < HD / 8; ++d) {
      dst[8 * d] = from_f32<T>(o[d][2 * r] * KT_DOWN * f);
      dst[8 * d + 1] = from_f32<T>(o[d][2 * r + 1] * KT_DOWN * f);
    }
  }
}

// the shares of a row joined: a block a (token, head), a thread a dim
template <typename T>
__global__ void kv8_tile_merge_kernel(const KtArgs a) {
  pdl_wait();
  pdl_trigger();
  const int token = blockIdx.x / a.nh, head = blockIdx.x % a.nh, d = threadIdx.x, hd = blockDim.x;
  const float2* ml = reinterpret_cast<const float2*>(a.part_ml) + (size_t)blockIdx.x * a.n_splits;
  const float* po = a.part_o + (size_t)blockIdx.x * a.n_splits * hd + d;
  const float sink = a.sinks ? a.sinks[head] * KT_LOG2E : -INFINITY;
  float top = sink;
  for (int i = 0; i < a.n_splits; ++i) top = fmaxf(top, ml[i].x);
  const float base = top == -INFINITY ? 0.f : top;
  float L = kv8_ex2(sink - base), O = 0.f;
#pragma unroll 4
  for (int i = 0; i < a.n_splits; ++i) {
    const float f = kv8_ex2(ml[i].x - base);
    L += ml[i].y * f;
    O += po[(size_t)i * hd] * f;
  }
  reinterpret_cast<T*>(a.out)[(size_t)token * a.out_stride + head * hd + d] = from_f32<T>(L == 0.f ? 0.f : O / L * a.out_scale);
}

template <typename T, int HD>
static int kt_launch(const KtArgs& a, int S, int n_tokens, cudaStream_t stream) {
  constexpr int SMEM = KT_STAGES * (2 * SX_PAGE * HD + 2 * SX_PAGE);
  static bool opted[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64 || !opted[dev]) {
    e = cudaFuncSetAttribute(kv8_tile_kernel<T, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    if (e != cudaSuccess) return (int)e;
    if (dev >= 0 && dev < 64) opted[dev] = true;
  }
  const int rc = sx_launch(kv8_tile_kernel<T, HD>, dim3((unsigned)a.n_tiles * a.n_splits, a.nkv, S), dim3(KT_WARPS * 32), SMEM, stream, a);
  if (rc || a.n_splits == 1) return rc;
  return sx_launch(kv8_tile_merge_kernel<T>, dim3((unsigned)n_tokens * a.nh), dim3(HD), 0, stream, a);
}

// `n_tokens` packed tokens of S sequences, no more than max_new of one.  Shares (`n_splits`) above 1 need part_o [n_tokens, nh, n_splits, hd] and
// part_ml [n_tokens, nh, n_splits, 2].
extern "C" int sx_kv8_tile(const void* q, void* out, const void* k, const void* v, const void* k_exp, const void* v_exp, const int* cu_seqlens,
                           const int* seq_past, const int* block_table, int maxp, int S, int n_tokens, int max_new, int nh, int nkv, int hd,
                           int n_pages, float scale, int window, float softcap, const float* sinks, int chunk, int out_stride, float out_scale,
                           int n_splits, float* part_o, float* part_ml, int dt, cudaStream_t stream) {
  if (S <= 0 || n_tokens <= 0) return 0;
  if ((hd != 64 && hd != 128) || nkv <= 0 || nkv > 65535 || nh <= 0 || nh % nkv || nh / nkv > KT_ROWS || S > 65535 || max_new < 1 || n_splits < 1 ||
      (n_splits > 1 && (!part_o || !part_ml)))
    return SX_ERR_SIZE;
  const int tokens = KT_ROWS / (nh / nkv), n_tiles = (max_new + tokens - 1) / tokens;
  if ((long long)n_tiles * n_splits > 0x7fffffff || (long long)n_tokens * nh > 0x7fffffff) return SX_ERR_SIZE;
  if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)k_exp | (uintptr_t)v_exp) & 15) return SX_ERR_ALIGN;
  const KtArgs a = {q, out, (const uint8_t*)k, (const uint8_t*)v, (const uint8_t*)k_exp, (const uint8_t*)v_exp, cu_seqlens, seq_past, block_table, sinks,
                    part_o, part_ml, maxp, n_pages, nh, nkv, window, chunk, out_stride, n_tiles, n_splits, scale, softcap, out_scale};
  if (dt == SX_F32) return hd == 64 ? kt_launch<float, 64>(a, S, n_tokens, stream) : kt_launch<float, 128>(a, S, n_tokens, stream);
  if (dt == SX_BF16) return hd == 64 ? kt_launch<bf16, 64>(a, S, n_tokens, stream) : kt_launch<bf16, 128>(a, S, n_tokens, stream);
  return SX_ERR_DTYPE;
}
