// Attention of few query rows over the 4-bit cache (single tokens, drafted
// tokens): qflash_kv4_attend's path for launches that the cache's bytes bound.
//
//   S_rj = scale * ks_j * sum_d q_rd (kc_jd - kz_j)      P = softmax(S)
//   O_rd = sum_j P_rj vs_j (vc_jd - vz_j)
//
// Scales stay outside the products: what the tensor cores multiply is the
// queries (as given) with whole numbers -15..15, exact in bf16 and fp16, and
// P vs with whole numbers.  P vs is rounded to bf16 once for bf16 queries
// (half a step, 2^-8, like the output's own rounding); for fp16 queries it is
// split into two bf16 terms (2^-16), since one would cost the output's last
// three bits.
//
// Both products are transposed, so that the cache is the MMA's A operand and is
// decoded straight into A fragments in registers, with no shared memory:
//   S^T = K Q^T: 16 keys x 8 rows per m16n8k16.  A thread (g, t) holds rows g
//     and g + 8 of K, and since the order of the reduction over d is free, it
//     loads one run of D / 8 bytes of its keys: the warp's loads are whole rows.
//   O^T = V^T P^T: 16 dims x 8 rows, reduced over keys.  Thread (g, t) holds
//     dims [g D/8, (g + 1) D/8) of keys 2t, 2t + 1 of each 8: two words of
//     neighbouring keys are interleaved with prmt, after which a half2 is
//     masked out of a word as in K's case.
// S^T's accumulator layout becomes P^T's B fragment by one 8x8 transpose
// (movmatrix) per 8 keys; rows of the softmax are columns here, so the maximum
// is taken over registers and 3 shuffles.
//
// Work split: (sequence, kv head, row tile) units are cut into tiles of 128
// keys, all tiles are numbered, and the CTAs of one resident wave each take an
// equal run of them (lengths are known on the device only).  A unit that one
// CTA holds whole is written by it; pieces go to the workspace with their
// maximum and sum, and a second kernel joins them in order.
#include <algorithm>

#include "kv4_common.cuh"

namespace qfb {
namespace kv4 {

constexpr int kTile = 128;        // keys per CTA tile: 4 warps of 32
constexpr int kWarps = 4;
constexpr int kRowsMax = 64;      // query rows (tokens x rep) per launch that accumulates weights

struct RowsArgs {
  AttendArgs a;
  int rows;       // ntok * rep
  int row_tiles;  // ceil(rows / (8 NT))
  int grid;       // CTAs of the first kernel
  int score_rows; // rows rounded up to even: the score buffer's row length
  float* parts;   // [grid][2][8 NT (D + 2)]: m, l, O of a piece
  float2* stats;  // [Z H row_tiles][8 NT]: m, l of units that one CTA held
  float* scores;  // [Z H][C][score_rows], in units of log2; null without weights
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_fp16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t y;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(y) : "f"(hi), "f"(lo));
  return y;
}
// Codes (low 4 bits of both halves) as numbers minus `zero`, exact: the code is
// set into the mantissa of 128 (bf16) or 1024 (fp16), `zero` is 128 (1024) + zero point.
template <bool FP16>
__device__ __forceinline__ uint32_t code_pair(uint32_t x, uint32_t zero) {
  const uint32_t m = (x & 0x000f000fu) | (FP16 ? 0x64006400u : 0x43004300u);
  uint32_t y;
  if (FP16)
    asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(m), "r"(zero));
  else
    asm("sub.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(m), "r"(zero));
  return y;
}

// Tiles of all units before sequence z, and of all sequences.  One warp.
__device__ __forceinline__ void tiles_before(const RowsArgs& p, int z, long long* before, long long* total) {
  const int lane = threadIdx.x & 31;
  const long long units = (long long)p.a.c.H * p.row_tiles;
  long long blo = 0, ball = 0;
  for (int i = lane; i < p.a.c.Z; i += 32) {
    const int t = (span_of(p.a, i).most(p.a) + kTile - 1) / kTile;
    ball += t;
    if (i < z) blo += t;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    ball += __shfl_xor_sync(~0u, ball, o);
    blo += __shfl_xor_sync(~0u, blo, o);
  }
  *before = blo * units;
  *total = ball * units;
}

// The sequence that holds tile `at`, and the number of its first tile.  One warp.
__device__ __forceinline__ int sequence_of(const RowsArgs& p, long long at, long long* first) {
  const int lane = threadIdx.x & 31;
  const long long units = (long long)p.a.c.H * p.row_tiles;
  long long base = 0;
  for (int z0 = 0; z0 < p.a.c.Z; z0 += 32) {
    const int i = z0 + lane;
    const long long mine = i < p.a.c.Z ? (long long)((span_of(p.a, i).most(p.a) + kTile - 1) / kTile) * units : 0;
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long up = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += up;
    }
    const unsigned hit = __ballot_sync(~0u, at >= base + sum - mine && at < base + sum);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *first = base + __shfl_sync(~0u, sum - mine, l);
      return z0 + l;
    }
    base += __shfl_sync(~0u, sum, 31);
  }
  *first = base;
  return p.a.c.Z;
}

__device__ __forceinline__ long long run_start(long long total, int grid, int cta) { return total * cta / grid; }

template <int D>
struct Raw {
  uint32_t k[4][D / 32];  // keys 8 i + g: D / 8 bytes each
  uint32_t v[8][D / 64];  // keys 8 (i / 2) + 2 t + (i & 1): D / 16 bytes each
  uint32_t kp, vp;        // parameters of key `lane`
};

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&r)[W], const uint8_t* p) {
  if constexpr (W == 4) {
    const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
    r[0] = x.x, r[1] = x.y, r[2] = x.z, r[3] = x.w;
  } else if constexpr (W == 2) {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
    r[0] = x.x, r[1] = x.y;
  } else {
    r[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
  }
}

// The 32 keys from key0 on; keys past `most` read the last one's codes (they are masked) and parameters 0.
template <int D>
__device__ __forceinline__ void load_tile(Raw<D>& r, const uint8_t* kc, const uint8_t* vc, const uint32_t* kp,
                                          const uint32_t* vp, int key0, int most) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    load_words<D / 32>(r.k[i], kc + (uint32_t)min(key0 + 8 * i + g, most - 1) * (D / 2u) + t * (D / 8));
#pragma unroll
  for (int i = 0; i < 8; ++i)
    load_words<D / 64>(r.v[i], vc + (uint32_t)min(key0 + 8 * (i >> 1) + 2 * t + (i & 1), most - 1) * (D / 2u) + g * (D / 16));
  const int key = key0 + lane;
  r.kp = key < most ? __ldg(kp + key) : 0u;
  r.vp = key < most ? __ldg(vp + key) : 0u;
}

template <int D, int NT, bool FP16>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 3 : 2) rows_kernel(RowsArgs p) {
  constexpr int R = 8 * NT;
  constexpr int kPad = D + 4;
  __shared__ float so[kWarps][R][kPad];
  __shared__ float sm[kWarps][R], sl[kWarps][R];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  long long before, total;
  tiles_before(p, 0, &before, &total);
  const int grid = (int)min((long long)p.grid, total);  // no CTA's run is empty
  if ((int)blockIdx.x >= grid) return;
  long long at = run_start(total, grid, blockIdx.x);
  const long long stop = run_start(total, grid, blockIdx.x + 1);
  long long zfirst;
  int z = sequence_of(p, at, &zfirst);
  if (z >= c.Z) return;  // only if lens changed meanwhile
  Span sp = span_of(a, z);
  int most = sp.most(a);
  int tiles = (most + kTile - 1) / kTile;
  int piece = 0;  // the first piece of a CTA goes to slot 0, a later cut one (its last) to slot 1
  const int units = c.H * p.row_tiles;
  while (at < stop) {
    long long in_z = at - zfirst;
    while (tiles == 0 || in_z >= (long long)units * tiles) {  // on to the next sequence that has tiles
      zfirst += (long long)units * tiles;
      in_z = at - zfirst;
      if (++z >= c.Z) return;
      sp = span_of(a, z);
      most = sp.most(a);
      tiles = (most + kTile - 1) / kTile;
    }
    const int unit = (int)(in_z / tiles), t0 = (int)(in_z % tiles);
    const int t1 = (int)min((long long)tiles, t0 + (stop - at));
    const int h = unit / p.row_tiles, row0 = (unit % p.row_tiles) * R;
    const size_t head = (size_t)z * c.H + h;
    const uint8_t* kc = c.codes[0] + head * c.C * (D / 2);
    const uint8_t* vc = c.codes[1] + head * c.C * (D / 2);
    const uint32_t* kp = c.param[0] + head * c.C;
    const uint32_t* vp = c.param[1] + head * c.C;

    // queries as B fragments, in the order of d that K's runs are loaded in
    uint32_t qf[NT][D / 16][2];
    int limit[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + 8 * n + g, tok = a.tok0 + row / a.rep;
      const bool live = row < p.rows && tok < sp.fresh;
      const uint16_t* q = (const uint16_t*)a.q + (live ? z * a.qs[0] + (h * a.rep + row % a.rep) * a.qs[1] + tok * a.qs[2] : 0);
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int d = t * (D / 4) + 8 * (s >> 1) + 2 * (s & 1) + j;
          qf[n][s][j] = live ? (uint32_t)__ldg(q + d) | ((uint32_t)__ldg(q + d + 4) << 16) : 0u;
        }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = row0 + 8 * n + 2 * t + j;
        limit[n][j] = r < p.rows ? sp.limit(a, a.tok0 + r / a.rep) : 0;
      }
    }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][i][j] = 0.f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
    }

    Raw<D> raw;
    load_tile<D>(raw, kc, vc, kp, vp, t0 * kTile + warp * 32, most);
    for (int tile = t0; tile < t1; ++tile) {
      const int key0 = tile * kTile + warp * 32;
      const Raw<D> cur = raw;
      if (tile + 1 < t1) load_tile<D>(raw, kc, vc, kp, vp, key0 + kTile, most);
      if (key0 >= most) continue;
      const float kscale = param_scale(cur.kp) * a.scale_log2e, vscale = param_scale(cur.vp);
      // zero points behind the offset that code_pair's numbers carry
      uint32_t kzero, vzero;
      {
        const float zk = param_zero(cur.kp), zv = param_zero(cur.vp);
        if (FP16) {
          const __half2 x = __float2half2_rn(1024.f + zk);
          kzero = *reinterpret_cast<const uint32_t*>(&x);
        } else {
          kzero = pack_bf16(128.f + zk, 128.f + zk);
        }
        const float other = __shfl_xor_sync(~0u, zv, 1);
        vzero = lane & 1 ? pack_bf16(128.f + other, 128.f + zv) : pack_bf16(128.f + zv, 128.f + other);
      }
      float s[NT][2][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const uint32_t z0 = __shfl_sync(~0u, kzero, 16 * mt + g), z1 = __shfl_sync(~0u, kzero, 16 * mt + 8 + g);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][mt][j] = 0.f;
#pragma unroll
        for (int st = 0; st < D / 16; ++st) {
          const uint32_t w0 = cur.k[2 * mt][st >> 1], w1 = cur.k[2 * mt + 1][st >> 1];
          const int sh = 8 * (st & 1);
          const uint32_t af[4] = {code_pair<FP16>(w0 >> sh, z0), code_pair<FP16>(w1 >> sh, z1),
                                  code_pair<FP16>(w0 >> (sh + 4), z0), code_pair<FP16>(w1 >> (sh + 4), z1)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (FP16)
              mma_fp16(s[n][mt], af, qf[n][st][0], qf[n][st][1]);
            else
              mma_bf16(s[n][mt], af, qf[n][st][0], qf[n][st][1]);
          }
        }
      }
      // scale, mask, running maximum
      float vs[4];
      bool moved = false;
      float mn[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) mn[n][0] = m[n][0], mn[n][1] = m[n][1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float ks = __shfl_sync(~0u, kscale, 8 * i + g);
        vs[i] = __shfl_sync(~0u, vscale, 8 * i + g);
        const int key = key0 + 8 * i + g;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float x[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            x[j] = s[n][i >> 1][2 * (i & 1) + j] * ks;
            if (key >= limit[n][j]) x[j] = -INFINITY;
            s[n][i >> 1][2 * (i & 1) + j] = x[j];
            mn[n][j] = fmaxf(mn[n][j], x[j]);
          }
          if (p.scores && key < most && row0 + 8 * n + 2 * t < p.rows)
            *reinterpret_cast<float2*>(p.scores + (head * c.C + key) * p.score_rows + row0 + 8 * n + 2 * t) = make_float2(x[0], x[1]);
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) mn[n][j] = fmaxf(mn[n][j], __shfl_xor_sync(~0u, mn[n][j], x));
          moved |= mn[n][j] > m[n][j];
        }
      if (__any_sync(~0u, moved)) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float f[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            f[j] = mn[n][j] == -INFINITY ? 1.f : ex2(m[n][j] - mn[n][j]);
            l[n][j] *= f[j];
            m[n][j] = mn[n][j];
          }
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            o[n][i][0] *= f[0], o[n][i][1] *= f[1];
            o[n][i][2] *= f[0], o[n][i][3] *= f[1];
          }
        }
      }
      float top[NT][2];  // a maximum of -inf (nothing seen yet, or scores of -inf alone) is no number to subtract
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) top[n][j] = m[n][j] == -INFINITY ? 0.f : m[n][j];
      // P vs as B fragments [keys of 8][rows]
      uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float y[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = s[n][i >> 1][2 * (i & 1) + j];
            const bool seen = key0 + 8 * i + g < limit[n][j];
            const float e = seen ? ex2(x - top[n][j]) : 0.f;
            l[n][j] += e;
            y[j] = seen ? e * vs[i] : 0.f;  // a masked position's scale may be anything
          }
          const uint32_t hi = pack_bf16(y[0], y[1]);
          ph[n][i] = transpose8(hi);
          if (FP16) {
            const uint32_t lo = pack_bf16(y[0] - __uint_as_float(hi << 16), y[1] - __uint_as_float(hi & 0xffff0000u));
            pl[n][i] = transpose8(lo);
          }
        }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const uint32_t z0 = __shfl_sync(~0u, vzero, 16 * ks + 2 * t), z1 = __shfl_sync(~0u, vzero, 16 * ks + 8 + 2 * t);
#pragma unroll
        for (int w = 0; w < D / 64; ++w) {
          // words of neighbouring keys, interleaved by halves
          uint32_t x[2][2];
#pragma unroll
          for (int b = 0; b < 2; ++b) {
            const uint32_t e = cur.v[4 * ks + 2 * b][w], f = cur.v[4 * ks + 2 * b + 1][w];
            x[b][0] = __byte_perm(e, f, 0x5410);
            x[b][1] = __byte_perm(e, f, 0x7632);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // dims 8 w + 2 i, 8 w + 2 i + 1 of this thread's run
            const int half = i >> 1, sh = 8 * (i & 1);
            const uint32_t af[4] = {code_pair<false>(x[0][half] >> sh, z0), code_pair<false>(x[0][half] >> (sh + 4), z0),
                                    code_pair<false>(x[1][half] >> sh, z1), code_pair<false>(x[1][half] >> (sh + 4), z1)};
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma_bf16(o[n][4 * w + i], af, ph[n][2 * ks], ph[n][2 * ks + 1]);
              if (FP16) mma_bf16(o[n][4 * w + i], af, pl[n][2 * ks], pl[n][2 * ks + 1]);
            }
          }
        }
      }
    }

    // join the 4 warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[n][j] += __shfl_xor_sync(~0u, l[n][j], x);
        const int r = 8 * n + 2 * t + j;
        if (g == 0) sm[warp][r] = m[n][j], sl[warp][r] = l[n][j];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          // accumulator rows g and g + 8 of m-tile i are dims 2 i and 2 i + 1 of run g
          so[warp][r][g * (D / 8) + 2 * i] = o[n][i][j];
          so[warp][r][g * (D / 8) + 2 * i + 1] = o[n][i][2 + j];
        }
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    float* part = p.parts + ((size_t)blockIdx.x * 2 + (piece ? 1 : 0)) * (R * (D + 2));
    for (int e = tid; e < R * D; e += kWarps * 32) {
      const int r = e / D, d = e % D, row = row0 + r;
      if (row >= p.rows) break;
      float mm = sm[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, sm[w][r]);
      float ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = sm[w][r] == -INFINITY ? 0.f : ex2(sm[w][r] - mm);
        // a warp that saw no key of this row holds l = 0 and O = 0; one that saw only NaN holds NaN
        ll += sm[w][r] == -INFINITY ? sl[w][r] : sl[w][r] * f;
        oo += sm[w][r] == -INFINITY ? so[w][r][d] : so[w][r][d] * f;
      }
      if (whole) {
        const int tok = a.tok0 + row / a.rep;
        const float y = sp.limit(a, tok) > 0 ? oo / ll : 0.f;
        const size_t at_out = z * a.os[0] + (h * a.rep + row % a.rep) * a.os[1] + tok * a.os[2] + d;
        if (FP16)
          ((__half*)a.out)[at_out] = __float2half_rn(y);
        else
          ((__nv_bfloat16*)a.out)[at_out] = __float2bfloat16_rn(y);
        if (d == 0 && p.scores) p.stats[(head * p.row_tiles + unit % p.row_tiles) * R + r] = make_float2(mm, ll);
      } else {
        part[2 * R + r * D + d] = oo;
        if (d == 0) part[r] = mm, part[R + r] = ll;
      }
    }
    __syncthreads();
    at += t1 - t0;
    ++piece;
  }
}

// Joins the pieces of units that several CTAs held, writes zeros for units with
// nothing to see, and adds the attention weights: blockIdx.x is a unit,
// blockIdx.y 0 its output, y > 0 a run of kChunk positions' weights.
constexpr int kChunk = 1024;

template <int D, int NT, bool FP16>
__global__ void __launch_bounds__(256) rows_finish_kernel(RowsArgs p) {
  constexpr int R = 8 * NT;
  constexpr int kPart = R * (D + 2);
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  const int rt = blockIdx.x % p.row_tiles, zh = blockIdx.x / p.row_tiles, z = zh / c.H, h = zh % c.H;
  const Span sp = span_of(a, z);
  const int most = sp.most(a), tiles = (most + kTile - 1) / kTile;
  const int tid = threadIdx.x;
  if (blockIdx.y > 0 && rt > 0) return;
  long long before = 0, total = 0;
  if (tiles) tiles_before(p, z, &before, &total);
  const int ctas = (int)min((long long)p.grid, total);

  // slot of the piece that CTA k holds of the unit whose first tile is `at`
  auto slot = [&](long long at, int k) { return 2 * k + (run_start(total, ctas, k) < at ? 1 : 0); };
  auto holder = [&](long long at) { return (int)min(ctas - 1LL, ((at + 1) * ctas - 1) / total); };

  if (blockIdx.y == 0) {
    const int row0 = rt * R, rows = min(R, p.rows - row0);
    int c0 = 0, c1 = 0;
    const long long at = before + ((long long)h * p.row_tiles + rt) * tiles;
    if (tiles) {
      c0 = holder(at), c1 = holder(at + tiles - 1);
      if (c0 == c1) return;  // written by its holder
    }
    for (int e = tid; e < rows * D; e += 256) {
      const int r = e / D, d = e % D, row = row0 + r, tok = a.tok0 + row / a.rep;
      float y = 0.f;
      if (tiles && sp.limit(a, tok) > 0) {
        float mm = -INFINITY, ll = 0.f, oo = 0.f;
        for (int k = c0; k <= c1; ++k) {
          const float* part = p.parts + (size_t)(k == c0 ? slot(at, k) : 2 * k) * kPart;
          const float pm = part[r], plv = part[R + r], po = part[2 * R + r * D + d];
          const float mx = fmaxf(mm, pm);
          const float f0 = mm == -INFINITY ? 1.f : ex2(mm - mx), f1 = pm == -INFINITY ? 1.f : ex2(pm - mx);
          ll = ll * f0 + plv * f1;
          oo = oo * f0 + po * f1;
          mm = mx;
        }
        y = oo / ll;
      }
      const size_t to = z * a.os[0] + (h * a.rep + row % a.rep) * a.os[1] + tok * a.os[2] + d;
      if (FP16)
        ((__half*)a.out)[to] = __float2half_rn(y);
      else
        ((__nv_bfloat16*)a.out)[to] = __float2bfloat16_rn(y);
    }
    return;
  }

  // weights: w_j += sum over rows of 2^(S_rj - m_r) / l_r
  const int j0 = (blockIdx.y - 1) * kChunk, j1 = min(sp.len, j0 + kChunk);
  if (j0 >= j1) return;
  __shared__ float sm[kRowsMax], sinv[kRowsMax];
  for (int row = tid; row < p.rows; row += 256) {
    float mm = -INFINITY, ll = 0.f;
    if (tiles && sp.limit(a, a.tok0 + row / a.rep) > 0) {
      const int u = row / R, r = row % R;
      const long long at = before + ((long long)h * p.row_tiles + u) * tiles;
      const int c0 = holder(at), c1 = holder(at + tiles - 1);
      if (c0 == c1) {
        const float2 s = p.stats[((size_t)zh * p.row_tiles + u) * R + r];
        mm = s.x, ll = s.y;
      } else {
        for (int k = c0; k <= c1; ++k) {
          const float* part = p.parts + (size_t)(k == c0 ? slot(at, k) : 2 * k) * kPart;
          const float pm = part[r], plv = part[R + r], mx = fmaxf(mm, pm);
          ll = ll * (mm == -INFINITY ? 1.f : ex2(mm - mx)) + plv * (pm == -INFINITY ? 1.f : ex2(pm - mx));
          mm = mx;
        }
      }
      sm[row] = mm, sinv[row] = 1.f / ll;
    } else {
      sm[row] = 0.f, sinv[row] = 0.f;
    }
  }
  __syncthreads();
  for (int j = j0 + tid; j < j1; j += 256) {
    float add = 0.f;
    if (j < most) {
      const float* s = p.scores + ((size_t)zh * c.C + j) * p.score_rows;
      for (int row = 0; row < p.rows; ++row) {
        const int lim = sp.limit(a, a.tok0 + row / a.rep);
        if (j < lim) add += ex2(s[row] - sm[row]) * sinv[row];
      }
    }
    const size_t w = (size_t)zh * c.C + j;
    c.weight[w] = a.weights_in[w] + add;
  }
}

// ------------------------------------------------------------------ host
static int tokens_per_launch(int rep, int N, bool weights) { return weights ? std::max(1, std::min(N, kRowsMax / rep)) : N; }

struct RowsPlan {
  int nt, row_tiles, rows, score_rows;
  long long parts, stats, scores;  // floats
};
constexpr int kGridMax = 148 * 3 * 2;

static RowsPlan plan_rows(const Cache& c, int rep, int ntok, bool weights) {
  RowsPlan p;
  p.rows = rep * ntok;
  p.nt = p.rows <= 8 ? 1 : 2;
  p.row_tiles = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
  p.score_rows = (p.rows + 1) / 2 * 2;
  p.parts = 2LL * kGridMax * 8 * p.nt * (c.D + 2);
  p.stats = weights ? 2LL * c.Z * c.H * p.row_tiles * 8 * p.nt : 0;
  p.scores = weights ? (long long)c.Z * c.H * c.C * p.score_rows : 0;
  return p;
}

size_t rows_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights) {
  const int rep = Hq / c->H, n = tokens_per_launch(rep, N, weights);
  const RowsPlan p = plan_rows(view(c), rep, n, weights);
  return (size_t)(p.parts + p.stats + p.scores) * 4;
}

template <int D, int NT, bool FP16>
static int launch_rows(RowsArgs r, int dev, cudaStream_t s) {
  const Cache& c = r.a.c;
  static int per_sm = 0;
  if (!per_sm) {
    int n = 0;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rows_kernel<D, NT, FP16>, kWarps * 32, 0) != cudaSuccess || n < 1)
      return set_err(QFLASH_ERR_LAUNCH, "kv4 rows: occupancy: %s", cudaGetErrorString(cudaGetLastError()));
    per_sm = n;
  }
  const long long tiles = (long long)c.Z * c.H * r.row_tiles * ((c.C + kTile - 1) / kTile);
  r.grid = (int)std::min<long long>(std::min<long long>((long long)sm_count(dev) * per_sm, kGridMax), tiles);
  rows_kernel<D, NT, FP16><<<r.grid, kWarps * 32, 0, s>>>(r);
  if (int rc = check_launch("kv4 rows", r.grid)) return rc;
  const dim3 grid(c.Z * c.H * r.row_tiles, r.scores ? 1 + (c.C + kChunk - 1) / kChunk : 1);
  rows_finish_kernel<D, NT, FP16><<<grid, 256, 0, s>>>(r);
  return check_launch("kv4 rows finish", grid.x);
}

int attend_rows(const AttendArgs& a0, bool fp16, void* ws, int dev, cudaStream_t s) {
  const bool weights = a0.weights_in != nullptr;
  const int step = tokens_per_launch(a0.rep, a0.N, weights);
  const RowsPlan most = plan_rows(a0.c, a0.rep, step, weights);
  for (int t0 = 0; t0 < a0.N; t0 += step) {
    RowsArgs r;
    r.a = a0;
    r.a.tok0 = t0;
    r.a.ntok = std::min(step, a0.N - t0);
    if (t0 && weights) r.a.weights_in = a0.c.weight;  // the launches before this one have added theirs
    const RowsPlan p = plan_rows(a0.c, a0.rep, r.a.ntok, weights);
    r.rows = p.rows;
    r.row_tiles = p.row_tiles;
    r.score_rows = p.score_rows;
    r.parts = (float*)ws;
    r.stats = (float2*)(r.parts + most.parts);
    r.scores = weights ? r.parts + most.parts + most.stats : nullptr;
    int rc;
    if (a0.c.D == 64)
      rc = p.nt == 1 ? (fp16 ? launch_rows<64, 1, true>(r, dev, s) : launch_rows<64, 1, false>(r, dev, s))
                     : (fp16 ? launch_rows<64, 2, true>(r, dev, s) : launch_rows<64, 2, false>(r, dev, s));
    else
      rc = p.nt == 1 ? (fp16 ? launch_rows<128, 1, true>(r, dev, s) : launch_rows<128, 1, false>(r, dev, s))
                     : (fp16 ? launch_rows<128, 2, true>(r, dev, s) : launch_rows<128, 2, false>(r, dev, s));
    if (rc) return rc;
  }
  return QFLASH_OK;
}

}  // namespace kv4
}  // namespace qfb
