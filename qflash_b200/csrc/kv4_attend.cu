// Attention of few query rows over the 4-bit cache (single tokens, drafted
// tokens): qflash_kv4_attend's path for launches that the cache's bytes bound.
//
//   S_rj = scale * ks_j * sum_d q_rd (kc_jd - kz_j)      P = softmax(S)
//   O_rd = sum_j P_rj vs_j (vc_jd - vz_j)
//
// Scales stay outside the products: what the tensor cores multiply is the
// queries (as given) with whole numbers -15..15, exact in bf16 and fp16, and
// P vs with whole numbers.  P vs is split into two bf16 terms (together 16 bits, off
// by 2^-16): bf16 because values' scales may lie anywhere in its range, two because one
// (2^-8) would cost fp16 outputs their last three bits, and bf16 outputs as much as their own
// rounding does (131071 positions: 0.0023 of the outputs' size against 0.0017).  The second
// term costs 10 % for bf16 queries (131071 positions 39.4 -> 43.3 us).
//
// Both products are transposed, so that the cache is the MMA's A operand, decoded
// straight into A fragments:
//   S^T = K Q^T: 16 keys x 8 rows per m16n8k16.  A thread (g, t) holds rows g
//     and g + 8 of K, and since the order of the reduction over d is free, it
//     reads one run of D / 8 bytes of its keys.
//   O^T = V^T P^T: 16 dims x 8 rows, reduced over keys.  ldmatrix.trans over
//     16-bit units of 4 codes leaves a thread with the units of keys 2t and
//     2t + 1 in the halves of a word: pairs of codes are masked out as in K's case.
// S^T's accumulator layout becomes P^T's B fragment by one 8x8 transpose
// (movmatrix) per 8 keys; rows of the softmax are columns here, so the maximum
// is taken over registers and 3 shuffles.
// Each warp has a ring of its own in shared memory, filled by cp.async two tiles
// ahead (a head's codes are contiguous), with 16-byte chunks swizzled against
// bank conflicts; no barrier but __syncwarp until the CTA's warps join.
//
// Work split: (sequence, kv head, row tile) units are cut into tiles of 128
// keys, all tiles are numbered, and the CTAs of one resident wave each take an
// equal run of them (lengths are known on the device only).  A unit that one
// CTA holds whole is written by it; pieces go to the workspace with their
// maximum and sum, and a second kernel joins them in order.  A unit counts for
// kBegin tiles more than it has, for its queries and its output: without that a CTA
// that got many units of a tile each was the last by far (16 ragged sequences of up to
// 4321, weights: 25.6 us; with 1, 2 and 4 tiles 21.0, 20.5 and 22.5).
//
// Measured, rows_kernel alone, head dim 128, bf16: 8 heads x 8 rows of 131071 positions
// (143 MB) 43 us, 3.3 TB/s; 32 ragged sequences of up to 8100 positions, 8 heads x 4 rows
// (196 MB), 57 us, 3.4 TB/s.  Arithmetic bounds it, most of it on codes: when P vs had one term the latter
// took 52 us, 40 without the masks and subtractions (a copy of the kernel), 52 without the MMAs, and the
// copies into shared memory alone take 26 of the former's 43.  55 % of issue slots are used, and warps that
// could issue wait for the arithmetic pipe as often as one issues.  A pair of codes costs one lop3 (the exponent comes
// with the mask, from a kernel argument that stays in a register), one subtraction, and for three pairs of
// four a shift.
// Registers are capped for 4 CTAs an SM (3 where 16 rows are held); ptxas then spills 36 bytes of stores for
// 8 rows of head dim 128, 16 for 8 rows of 64, and 336 for 16 rows of 128.
#include <algorithm>
#include <atomic>
#include <climits>

#include "kv4_common.cuh"

namespace qfb {
namespace kv4 {

constexpr int kTile = 128;        // keys per CTA tile: 4 warps of 32
constexpr int kWarps = 4;
constexpr int kGridMax = 148 * 5;  // CTAs of one resident wave at most

struct RowsArgs {
  AttendArgs a;
  int rows;       // N * rep
  int row_tiles;  // ceil(rows / (8 NT))
  int grid;       // CTAs of the first kernel
  uint32_t magic_k, magic_v;
  bool single;    // a CTA per unit, no second kernel
  bool vec_q;     // query rows start on 16-byte boundaries
  int score_rows; // 2, or rows rounded up to fours: the score buffer's row length
  float* parts;   // [grid][2][8 NT (D + 2)]: m, l, O of a piece
  float2* stats;  // [Z H row_tiles][8 NT]: m, l of units that one CTA held
  float* scores;  // [Z H][C][score_rows] of a launch's sequences and heads, in units of log2; null without weights
};

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
// Codes (low 4 bits of both halves) as numbers minus `zero`, exact: the code is
// set into the mantissa of 128 (bf16) or 1024 (fp16), `zero` is 128 (1024) +
// zero point.  `magic`, 128 or 1024 twice, comes from the kernel's arguments: as
// a known constant it and the mask became an instruction each (lop3 takes one
// immediate), and the integer pipe is what bounds this kernel.
template <bool FP16>
__device__ __forceinline__ uint32_t code_pair(uint32_t x, uint32_t magic, uint32_t zero) {
  uint32_t m, y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(m) : "r"(x), "r"(0x000f000fu), "r"(magic));  // (x & mask) | magic
  if (FP16)
    asm("sub.f16x2 %0, %1, %2;" : "=r"(y) : "r"(m), "r"(zero));
  else
    asm("sub.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(m), "r"(zero));
  return y;
}

// A unit of a sequence that shows `most` positions: its tiles, and what it counts for.
__device__ __forceinline__ int tiles_of(int most) { return (most + kTile - 1) / kTile; }
__device__ __forceinline__ int unit_cost(int most) { return cost_of(tiles_of(most)); }

// The cost of all units before sequence z, and of all sequences.  One warp.
__device__ __forceinline__ void cost_before(const RowsArgs& p, int z, long long* before, long long* total) {
  const int lane = threadIdx.x & 31;
  const long long units = (long long)p.a.c.H * p.row_tiles;
  long long blo = 0, ball = 0;
  for (int i = lane; i < p.a.c.Z; i += 32) {
    const int t = unit_cost(span_of(p.a, i).most(p.a));
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

// The sequence that holds place `at`, and where it begins.  One warp.
__device__ __forceinline__ int sequence_of(const RowsArgs& p, long long at, long long* first) {
  const int lane = threadIdx.x & 31;
  const long long units = (long long)p.a.c.H * p.row_tiles;
  long long base = 0;
  for (int z0 = 0; z0 < p.a.c.Z; z0 += 32) {
    const int i = z0 + lane;
    const long long mine = i < p.a.c.Z ? (long long)unit_cost(span_of(p.a, i).most(p.a)) * units : 0;
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

// What both give for the place a CTA's run begins at, lengths loaded once where
// one warp holds them all.  `place_of`: the run's beginning from the total.
struct Place {
  long long total, at, first;  // first: where sequence z begins
  int z, grid;
};
__device__ __forceinline__ Place begin_of(const RowsArgs& p, int cta) {
  Place r;
  const int lane = threadIdx.x & 31;
  if (p.a.c.Z > 32) {
    long long before;
    cost_before(p, 0, &before, &r.total);
    r.grid = (int)min((long long)p.grid, r.total);
    r.at = r.grid ? r.total * min(cta, r.grid) / r.grid : 0;
    r.z = cta < r.grid ? sequence_of(p, r.at, &r.first) : p.a.c.Z;
    return r;
  }
  const long long mine = lane < p.a.c.Z ? (long long)unit_cost(span_of(p.a, lane).most(p.a)) * p.a.c.H * p.row_tiles : 0;
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(~0u, sum, o);
    if (lane >= o) sum += up;
  }
  r.total = __shfl_sync(~0u, sum, 31);
  r.grid = (int)min((long long)p.grid, r.total);  // no CTA's run is empty
  r.at = r.grid ? r.total * min(cta, r.grid) / r.grid : 0;
  const unsigned hit = __ballot_sync(~0u, r.at >= sum - mine && r.at < sum);
  r.z = hit ? __ffs(hit) - 1 : p.a.c.Z;
  r.first = __shfl_sync(~0u, sum - mine, r.z & 31);
  return r;
}

__device__ __forceinline__ long long run_start(long long total, int grid, int cta) { return total * cta / grid; }

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {  // zeros where nothing is there
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A warp's stage: 32 keys' codes, values' codes, and both parameter words.
template <int D>
struct Stage {
  static constexpr int ROW = D / 2, CHUNKS = ROW / 16;
  static constexpr uint32_t K = 0, V = 32 * ROW, KP = 64 * ROW, VP = KP + 128, BYTES = VP + 128;
  static constexpr int COUNT = D == 128 ? 3 : 4;
  // row r's 16-byte chunk c lies at chunk c ^ turn(r): 8 rows' chunks c cover all banks
  __device__ static int turn(int r) { return D == 128 ? (r >> 1) & 3 : (r >> 2) & 1; }
};
constexpr int kJoinPad = 4;
template <int D, int NT>
constexpr uint32_t rows_smem() {
  constexpr uint32_t ring = kWarps * Stage<D>::COUNT * Stage<D>::BYTES, join = kWarps * 8 * NT * (D + kJoinPad) * 4;
  return ring > join ? ring : join;
}

// Where a lane's share of a warp's stages comes from; advanced tile by tile.
template <int D>
struct Source {
  const uint8_t *kc, *vc;      // 16 bytes per lane and chunk step
  const uint32_t *kp, *vp;     // one word per lane
};

// Starts the copy of the next 32 keys, `left` of which are there; zeros for the others.
template <int D>
__device__ __forceinline__ void fetch(uint32_t stage, Source<D>& src, int left) {
  using S = Stage<D>;
  const int lane = threadIdx.x & 31, r = lane / S::CHUNKS, c = lane % S::CHUNKS;
  const uint32_t to = stage + r * S::ROW + ((c ^ S::turn(r)) << 4);  // the turn is the same 8 and 16 rows on
  if (left >= 32) {
#pragma unroll
    for (int i = 0; i < S::CHUNKS; ++i) {
      copy_async<16>(to + S::K + i * 512, src.kc + i * 512, true);
      copy_async<16>(to + S::V + i * 512, src.vc + i * 512, true);
    }
    copy_async<4>(stage + S::KP + 4 * lane, src.kp, true);
    copy_async<4>(stage + S::VP + 4 * lane, src.vp, true);
  } else if (left > 0) {
#pragma unroll
    for (int i = 0; i < S::CHUNKS; ++i) {
      const bool there = r + i * (32 / S::CHUNKS) < left;
      const int step = there ? i * 512 : -(lane * 16);  // the tile's first bytes, of which nothing is read
      copy_async<16>(to + S::K + i * 512, src.kc + step, there);
      copy_async<16>(to + S::V + i * 512, src.vc + step, there);
    }
    const bool there = lane < left;
    copy_async<4>(stage + S::KP + 4 * lane, src.kp - (there ? 0 : lane), there);
    copy_async<4>(stage + S::VP + 4 * lane, src.vp - (there ? 0 : lane), there);
  }
  src.kc += kTile * S::ROW, src.vc += kTile * S::ROW;
  src.kp += kTile, src.vp += kTile;
}

template <int D, int NT, bool FP16>
struct RowsState {
  uint32_t q[NT][D / 16][2];  // queries as B fragments, in the order of d that K's runs are read in
  int limit[NT][2];           // positions that rows 2t, 2t + 1 of each 8 see
  float o[NT][D / 16][4], m[NT][2], l[NT][2];
};

// One stage of 32 keys.  FULL: every row sees all of them.
template <int D, int NT, bool FP16, bool FULL>
__device__ __forceinline__ void rows_step(RowsState<D, NT, FP16>& st, uint32_t stage, int key0, int most, float scale_log2e,
                                          uint32_t mk, uint32_t mv, float* scores, int score_rows, int rows_left) {
  using S = Stage<D>;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t kpw, vpw;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(kpw) : "r"(stage + S::KP + 4 * lane));
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(vpw) : "r"(stage + S::VP + 4 * lane));
  const float kscale = param_scale(kpw) * scale_log2e, vscale = param_scale(vpw);
  // zero points behind the offset that code_pair's numbers carry
  uint32_t kzero, vzero;
  {
    const float zk = param_zero(kpw), zv = param_zero(vpw);
    if (FP16) {
      const __half2 x = __float2half2_rn(1024.f + zk);
      kzero = *reinterpret_cast<const uint32_t*>(&x);
    } else {
      kzero = pack_bf16(128.f + zk, 128.f + zk);
    }
    const float other = __shfl_down_sync(~0u, zv, 1);
    vzero = pack_bf16(128.f + zv, 128.f + other);  // read from even lanes
  }
  float s[NT][2][4];
#pragma unroll
  for (int mt = 0; mt < 2; ++mt) {
    const uint32_t z0 = __shfl_sync(~0u, kzero, 16 * mt + g), z1 = __shfl_sync(~0u, kzero, 16 * mt + 8 + g);
    uint32_t k0[D / 32], k1[D / 32];
    const uint32_t at = stage + S::K + (16 * mt + g) * S::ROW +
                        (D == 128 ? (t ^ S::turn(g)) << 4 : (((t >> 1) ^ S::turn(g)) << 4) + (t & 1) * 8);
    if constexpr (D == 128) {
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(k0[0]), "=r"(k0[1]), "=r"(k0[2]), "=r"(k0[3]) : "r"(at));
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(k1[0]), "=r"(k1[1]), "=r"(k1[2]), "=r"(k1[3]) : "r"(at + 8 * S::ROW));
    } else {
      asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(k0[0]), "=r"(k0[1]) : "r"(at));
      asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(k1[0]), "=r"(k1[1]) : "r"(at + 8 * S::ROW));
    }
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[n][mt][j] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint32_t w0 = k0[i >> 1], w1 = k1[i >> 1];
      const int sh = 8 * (i & 1);
      const uint32_t af[4] = {code_pair<FP16>(w0 >> sh, mk, z0), code_pair<FP16>(w1 >> sh, mk, z1),
                              code_pair<FP16>(w0 >> (sh + 4), mk, z0), code_pair<FP16>(w1 >> (sh + 4), mk, z1)};
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        if (FP16)
          mma_fp16(s[n][mt], af, st.q[n][i][0], st.q[n][i][1]);
        else
          mma_bf16(s[n][mt], af, st.q[n][i][0], st.q[n][i][1]);
      }
    }
  }
  // Scale and mask.  O is rescaled only when a score exceeds its row's maximum so far by more than 8 (in log2):
  // P is at most 256 else, which costs no bits in floating point, and only then is the maximum formed over threads.
  float vs[4], mn[NT][2];
#pragma unroll
  for (int n = 0; n < NT; ++n) mn[n][0] = mn[n][1] = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float ks = __shfl_sync(~0u, kscale, 8 * i + g);
    vs[i] = __shfl_sync(~0u, vscale, 8 * i + g);
    const int key = key0 + 8 * i + g;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float* x = s[n][i >> 1] + 2 * (i & 1);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[j] *= ks;
        if (!FULL && key >= st.limit[n][j]) x[j] = -INFINITY;
      }
      if (scores && key < most && 8 * n + 2 * t < rows_left)
        *reinterpret_cast<float2*>(scores + (size_t)key * score_rows + 8 * n + 2 * t) = make_float2(x[0], x[1]);
    }
  }
  bool moved = false;
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mn[n][j] = max3(fmaxf(s[n][0][j], s[n][0][2 + j]), s[n][1][j], s[n][1][2 + j]);
      moved |= mn[n][j] > st.m[n][j] + 8.f;
    }
  if (__any_sync(~0u, moved)) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {  // all rows are brought up to date when one has to be
        mn[n][j] = fmaxf(mn[n][j], st.m[n][j]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) mn[n][j] = fmaxf(mn[n][j], __shfl_xor_sync(~0u, mn[n][j], x));
        f[j] = mn[n][j] == -INFINITY ? 1.f : ex2(st.m[n][j] - mn[n][j]);
        st.l[n][j] *= f[j];
        st.m[n][j] = mn[n][j];
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        st.o[n][i][0] *= f[0], st.o[n][i][1] *= f[1];
        st.o[n][i][2] *= f[0], st.o[n][i][3] *= f[1];
      }
    }
  }
  // P vs as B fragments [keys of 8][rows], the first terms and the second ones
  uint32_t ph[NT][4], pl[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float top[2];  // a maximum of -inf (nothing seen yet, or scores of -inf alone) is no number to subtract
#pragma unroll
    for (int j = 0; j < 2; ++j) top[j] = st.m[n][j] == -INFINITY ? 0.f : st.m[n][j];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float y[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float e = ex2(s[n][i >> 1][2 * (i & 1) + j] - top[j]);
        st.l[n][j] += e;
        y[j] = e * vs[i];
        if (!FULL && key0 + 8 * i + g >= st.limit[n][j]) y[j] = 0.f;  // a masked position's scale may be anything
      }
      const uint32_t hi = pack_bf16(y[0], y[1]);
      ph[n][i] = transpose8(hi);
      pl[n][i] = transpose8(pack_bf16(y[0] - __uint_as_float(hi << 16), y[1] - __uint_as_float(hi & 0xffff0000u)));
    }
  }
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    const uint32_t z0 = __shfl_sync(~0u, vzero, 16 * ks + 2 * t), z1 = __shfl_sync(~0u, vzero, 16 * ks + 8 + 2 * t);
    // matrices of an x4: keys 0-7 and 8-15 of dims 32 seg .., the same of the next 32 dims
    const int key = 16 * ks + 8 * (lane >> 3 & 1) + (lane & 7);
#pragma unroll
    for (int seg = 0; seg < D / 32; seg += 2) {
      uint32_t x[4];
      const uint32_t at = stage + S::V + key * S::ROW + (((seg + (lane >> 4)) ^ S::turn(lane & 7)) << 4);
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                   : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(at));
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // dims 32 (seg + i / 2) + 4 g + 2 (i & 1), and the next
        const uint32_t a = x[i & 2], b = x[(i & 2) + 1];
        const int sh = 8 * (i & 1);
        const uint32_t af[4] = {code_pair<false>(a >> sh, mv, z0), code_pair<false>(a >> (sh + 4), mv, z0),
                                code_pair<false>(b >> sh, mv, z1), code_pair<false>(b >> (sh + 4), mv, z1)};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma_bf16(st.o[n][2 * seg + i], af, ph[n][2 * ks], ph[n][2 * ks + 1]);
          mma_bf16(st.o[n][2 * seg + i], af, pl[n][2 * ks], pl[n][2 * ks + 1]);
        }
      }
    }
  }
}

template <int D, int NT, bool FP16>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 ? 4 : 3) rows_kernel(RowsArgs p) {
  using S = Stage<D>;
  constexpr int R = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  float(*so)[R][D + kJoinPad] = reinterpret_cast<float(*)[R][D + kJoinPad]>(smem);  // over the rings, when they are done
  __shared__ float sm[kWarps][R], sl[kWarps][R];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t ring = shared_addr(smem) + warp * (S::COUNT * S::BYTES);
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  may_begin();
  long long at, stop, zfirst;
  int z;
  if (p.single) {  // one unit, whole
    z = blockIdx.x / (c.H * p.row_tiles);
    zfirst = 0;
  } else {
    const Place me = begin_of(p, blockIdx.x);
    if ((int)blockIdx.x >= me.grid || me.z >= c.Z) return;  // the latter only if lens changed meanwhile
    at = me.at, zfirst = me.first, z = me.z;
    stop = run_start(me.total, me.grid, blockIdx.x + 1);
  }
  Span sp = span_of(a, z);
  int most = sp.most(a);
  int piece = 0;  // the first piece of a CTA goes to slot 0, a later cut one (its last) to slot 1
  const int units = c.H * p.row_tiles;
  if (p.single) {
    const int cost = unit_cost(most);
    at = (long long)(blockIdx.x % units) * cost, stop = at + cost;
    if (most <= 0) {  // nothing to see
      const int row0 = (int)(blockIdx.x % p.row_tiles) * R, h = (int)(blockIdx.x % units) / p.row_tiles;
      for (int e = tid; e < R * D; e += kWarps * 32) {
        const int row = row0 + e / D;
        if (row >= p.rows) break;
        const size_t to = z * a.os[0] + (h * a.rep + row % a.rep) * a.os[1] + (row / a.rep) * a.os[2] + e % D;
        ((uint16_t*)a.out)[to] = 0;
      }
      if (p.scores) {
        const size_t head = (size_t)z * c.H + h;
        for (int j = tid; j < sp.len; j += kWarps * 32) c.weight[head * c.C + j] = a.weights_in[head * c.C + j];
      }
      return;
    }
  }
  while (at < stop) {
    long long in_z = at - zfirst;
    while (most <= 0 || in_z >= (long long)units * unit_cost(most)) {  // on to the next sequence that shows anything
      zfirst += (long long)units * unit_cost(most);
      in_z = at - zfirst;
      if (++z >= c.Z) return;
      sp = span_of(a, z);
      most = sp.most(a);
    }
    const int tiles = tiles_of(most), cost = unit_cost(most);
    const int unit = (int)(in_z / cost), u0 = (int)(in_z % cost);  // kBegin places, then the tiles
    const int u1 = (int)min((long long)cost, u0 + (stop - at)), t0 = max(0, u0 - kBegin), t1 = u1 - kBegin;
    at += u1 - u0;
    if (t1 <= t0) continue;
    const int h = unit / p.row_tiles, row0 = (unit % p.row_tiles) * R;
    const size_t head = (size_t)z * c.H + h;
    const uint8_t* kc = c.codes[0] + head * c.C * (D / 2);
    const uint8_t* vc = c.codes[1] + head * c.C * (D / 2);
    const uint32_t* kp = c.param[0] + head * c.C;
    const uint32_t* vp = c.param[1] + head * c.C;

    const int first_key = t0 * kTile + warp * 32;
    Source<D> src = {kc + (size_t)first_key * S::ROW + lane * 16, vc + (size_t)first_key * S::ROW + lane * 16,
                     kp + first_key + lane, vp + first_key + lane};
    const int end = min(most, t1 * kTile);
    int fetched = first_key, to_stage = 0;
    auto start = [&] {
      fetch<D>(ring + to_stage * S::BYTES, src, end - fetched);
      copies_commit();
      fetched += kTile;
      to_stage = to_stage + 1 == S::COUNT ? 0 : to_stage + 1;
    };
#pragma unroll
    for (int i = 0; i < S::COUNT - 1; ++i) start();

    RowsState<D, NT, FP16> st;
    int least = INT_MAX;  // positions that every row sees
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int row = row0 + 8 * n + g, tok = row / a.rep;
      const bool live = row < p.rows && tok < sp.fresh;
      const uint16_t* q = (const uint16_t*)a.q + (live ? z * a.qs[0] + (h * a.rep + row % a.rep) * a.qs[1] + tok * a.qs[2] : 0) + t * (D / 4);
#pragma unroll
      for (int s = 0; s < D / 16; s += 2) {  // 8 elements: pairs d, d + 4
        uint4 x = make_uint4(0, 0, 0, 0);
        if (live && p.vec_q) {
          x = __ldg(reinterpret_cast<const uint4*>(q + 4 * s));
        } else if (live) {
          const uint16_t* e = q + 4 * s;
          x = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16, e[6] | (uint32_t)e[7] << 16);
        }
        st.q[n][s][0] = __byte_perm(x.x, x.z, 0x5410), st.q[n][s][1] = __byte_perm(x.x, x.z, 0x7632);
        st.q[n][s + 1][0] = __byte_perm(x.y, x.w, 0x5410), st.q[n][s + 1][1] = __byte_perm(x.y, x.w, 0x7632);
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = row0 + 8 * n + 2 * t + j, tk = r / a.rep;
        // rows that are not there see everything: nothing of them is used, and they must not keep the others from FULL
        st.limit[n][j] = r < p.rows && tk < sp.fresh ? sp.limit(a, tk) : INT_MAX;
        least = min(least, st.limit[n][j]);
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) st.o[n][i][j] = 0.f;
      st.m[n][0] = st.m[n][1] = -INFINITY;
      st.l[n][0] = st.l[n][1] = 0.f;
    }
    least = min(most, __reduce_min_sync(~0u, least));
    float* scores = p.scores ? p.scores + head * c.C * p.score_rows + row0 : nullptr;

    int at_stage = 0;
    for (int tile = t0; tile < t1; ++tile) {
      copies_wait<S::COUNT - 2>();
      __syncwarp();  // this tile's copies are there for all lanes, and all have left the stage that is filled next
      start();
      const int key0 = tile * kTile + warp * 32;
      const uint32_t stage = ring + at_stage * S::BYTES;
      at_stage = at_stage + 1 == S::COUNT ? 0 : at_stage + 1;
      if (key0 + 32 <= least)
        rows_step<D, NT, FP16, true>(st, stage, key0, most, a.scale_log2e, p.magic_k, p.magic_v, scores, p.score_rows, p.rows - row0);
      else if (key0 < most)
        rows_step<D, NT, FP16, false>(st, stage, key0, most, a.scale_log2e, p.magic_k, p.magic_v, scores, p.score_rows, p.rows - row0);
    }
    copies_wait<0>();
    __syncthreads();

    // join the 4 warps
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) st.l[n][j] += __shfl_xor_sync(~0u, st.l[n][j], x);
        const int r = 8 * n + 2 * t + j;
        if (g == 0) sm[warp][r] = st.m[n][j], sl[warp][r] = st.l[n][j];
#pragma unroll
        for (int i = 0; i < D / 16; ++i)  // accumulator rows g and g + 8
          *reinterpret_cast<float2*>(&so[warp][r][32 * (i >> 1) + 4 * g + 2 * (i & 1)]) = make_float2(st.o[n][i][j], st.o[n][i][2 + j]);
      }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == tiles;
    float* part = p.parts + ((size_t)blockIdx.x * 2 + (piece ? 1 : 0)) * (R * (D + 2));
    for (int e = tid; e < R * (D / 4); e += kWarps * 32) {
      const int r = e / (D / 4), d = e % (D / 4) * 4, row = row0 + r;
      if (row >= p.rows) break;
      float mm = sm[0][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, sm[w][r]);
      float ll = 0.f;
      float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        // a warp that saw no key of this row holds l = 0 and O = 0; one that saw only NaN holds NaN
        const float f = sm[w][r] == -INFINITY ? 1.f : ex2(sm[w][r] - mm);
        const float4 x = *reinterpret_cast<const float4*>(&so[w][r][d]);
        ll += sl[w][r] * f;
        oo.x += x.x * f, oo.y += x.y * f, oo.z += x.z * f, oo.w += x.w * f;
      }
      if (whole) {
        const int tok = row / a.rep;
        const bool seen = sp.limit(a, tok) > 0;
        const float inv = 1.f / ll, y[4] = {seen ? oo.x * inv : 0.f, seen ? oo.y * inv : 0.f, seen ? oo.z * inv : 0.f, seen ? oo.w * inv : 0.f};
        const size_t to = z * a.os[0] + (h * a.rep + row % a.rep) * a.os[1] + tok * a.os[2] + d;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (FP16)
            ((__half*)a.out)[to + i] = __float2half_rn(y[i]);
          else
            ((__nv_bfloat16*)a.out)[to + i] = __float2bfloat16_rn(y[i]);
        }
        if (d == 0 && p.scores && !p.single) p.stats[(head * p.row_tiles + unit % p.row_tiles) * R + r] = make_float2(mm, ll);
      } else {
        *reinterpret_cast<float4*>(part + 2 * R + r * D + d) = oo;
        if (d == 0) part[r] = mm, part[R + r] = ll;
      }
    }
    __syncthreads();
    ++piece;
    if (p.single && p.scores) {  // weights of a head that is this CTA's alone: its scores are behind the barriers above
      if (tid < R) {
        float mm = sm[0][tid], ll = 0.f;
#pragma unroll
        for (int w = 1; w < kWarps; ++w) mm = fmaxf(mm, sm[w][tid]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) ll += sl[w][tid] * (sm[w][tid] == -INFINITY ? 1.f : ex2(sm[w][tid] - mm));
        const int tok = tid / a.rep;
        const bool seen = tid < p.rows && sp.limit(a, tok) > 0;
        so[0][tid][0] = mm == -INFINITY ? 0.f : mm, so[0][tid][1] = seen ? 1.f / ll : 0.f;
        so[0][tid][2] = __int_as_float(seen ? sp.limit(a, tok) : 0);
      }
      __syncthreads();
      const float* s = p.scores + head * c.C * p.score_rows;
      for (int j = tid; j < sp.len; j += kWarps * 32) {
        float add = 0.f;
        if (j < most)
          for (int row = 0; row < p.rows; ++row)
            if (j < __float_as_int(so[0][row][2])) add += ex2(s[(size_t)j * p.score_rows + row] - so[0][row][0]) * so[0][row][1];
        c.weight[head * c.C + j] = a.weights_in[head * c.C + j] + add;
      }
    }
  }
}

// Begins while rows_kernel ends, adds about 6 us to a call, and 10 where it adds up weights:
// bound by the latency of its chain of loads (lengths, the pieces' statistics, pieces).
// Four rows' scores come in one load, and limits are taken out of the loop over positions: with
// scalar loads and a division per row, 32 rows over 8 heads of 4000 positions took 62 us in all,
// now 34.
// Joins the pieces of units that several CTAs held and writes zeros for units
// with nothing to see (a block per row of a unit), and adds the attention
// weights (the blocks behind them: kChunk positions of a head each).
constexpr int kChunk = 1024;
constexpr int kJoin = 256;  // threads

// The scores of 4 rows (2, if there are no more) from the first one's.
__device__ __forceinline__ float4 scores_of(const float* s, int score_rows) {
  if (score_rows > 2) return *reinterpret_cast<const float4*>(s);
  const float2 x = *reinterpret_cast<const float2*>(s);
  return make_float4(x.x, x.y, 0.f, 0.f);
}
constexpr int kPer = (kGridMax + kJoin - 1) / kJoin;

template <int D, int NT, bool FP16>
__global__ void __launch_bounds__(kJoin) rows_finish_kernel(RowsArgs p) {
  constexpr int R = 8 * NT;
  constexpr int kPart = R * (D + 2);
  __shared__ float sf[kGridMax];
  __shared__ float red[kJoin / 32], sums[kJoin];
  __shared__ __align__(16) float sm[kWeightRows], sinv[kWeightRows];
  __shared__ __align__(16) int seen_to[kWeightRows];
  const AttendArgs& a = p.a;
  const Cache& c = a.c;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // one block at least waits, whatever it has to do: the kernels behind this one go by its end
  if (blockIdx.x == 0) wait_for_previous();
  const int joins = c.Z * c.H * p.rows;
  const bool weigh = (int)blockIdx.x >= joins;
  const int chunks = (c.C + kChunk - 1) / kChunk;
  const int zh = weigh ? (blockIdx.x - joins) / chunks : blockIdx.x / p.rows, z = zh / c.H, h = zh % c.H;
  const Span sp = span_of(a, z);
  const int most = sp.most(a), tiles = tiles_of(most), cost = unit_cost(most);
  long long before = 0, total = 0;
  if (tiles) cost_before(p, z, &before, &total);
  const int ctas = (int)min((long long)p.grid, total);
  // The CTA that holds a place; and where CTA k's piece of a unit that begins at `first` is, c0 its first holder
  auto holder = [&](long long place) { return (int)min(ctas - 1LL, ((place + 1) * ctas - 1) / total); };
  auto part_of = [&](long long first, int c0, int k) {
    return p.parts + (size_t)(k == c0 && run_start(total, ctas, k) < first ? 2 * k + 1 : 2 * k) * kPart;
  };

  if (!weigh) {
    const int row = blockIdx.x % p.rows, u = row / R, r = row % R, tok = row / a.rep;
    const size_t to = z * a.os[0] + (h * a.rep + row % a.rep) * a.os[1] + tok * a.os[2];
    const bool seen = sp.limit(a, tok) > 0;
    const long long first = before + ((long long)h * p.row_tiles + u) * cost;
    const int c0 = tiles ? holder(first + kBegin) : 0, n = tiles ? holder(first + cost - 1) - c0 + 1 : 0;
    if (n == 1) return;  // written by its holder
    constexpr int G = kJoin / D;  // groups of threads that share a row's pieces
    constexpr int kAhead = 4;     // pieces whose part of O is on its way before the maximum is known
    const int d = tid % D, group = tid / D;
    float y = 0.f;
    wait_for_previous();
    if (seen) {
      auto piece = [&](int k) { return part_of(first, c0, c0 + k); };
      float pre[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) pre[i] = group + i * G < n ? piece(group + i * G)[2 * R + r * D + d] : 0.f;
      float pm[kPer], pl[kPer], mx = -INFINITY;  // this thread's pieces: tid, tid + kJoin ..
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int k = tid + i * kJoin;
        pm[i] = k < n ? piece(k)[r] : -INFINITY;
        pl[i] = k < n ? piece(k)[R + r] : 0.f;
        mx = fmaxf(mx, pm[i]);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
      if (lane == 0) red[warp] = mx;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kJoin / 32; ++w) mx = fmaxf(mx, red[w]);
      float l = 0.f;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const float f = pm[i] == -INFINITY ? 1.f : ex2(pm[i] - mx);
        if (tid + i * kJoin < n) sf[tid + i * kJoin] = f;
        l += f * pl[i];
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
      if (lane == 0) sums[warp] = l;
      __syncthreads();
      l = 0.f;
#pragma unroll
      for (int w = 0; w < kJoin / 32; ++w) l += sums[w];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        if (group + i * G < n) y += sf[group + i * G] * pre[i];
      // all but the first piece lie in their CTAs' slot 0
      const float* part = p.parts + (size_t)2 * c0 * kPart + 2 * R + r * D + d;
#pragma unroll 8
      for (int k = group + kAhead * G; k < n; k += G) y += sf[k] * part[(size_t)2 * k * kPart];
      sums[tid] = y;
      __syncthreads();
#pragma unroll
      for (int q = 1; q < G; ++q) y += sums[q * D + d];
      y /= l;
    }
    if (group == 0) {
      if (FP16)
        ((__half*)a.out)[to + d] = __float2half_rn(y);
      else
        ((__nv_bfloat16*)a.out)[to + d] = __float2bfloat16_rn(y);
    }
    return;
  }

  // weights: w_j += sum over rows of 2^(S_rj - m_r) / l_r
  const int j0 = (blockIdx.x - joins) % chunks * kChunk, j1 = min(sp.len, j0 + kChunk);
  if (j0 >= j1) return;
  constexpr int kKeysPer = kChunk / kJoin;
  float old[kKeysPer];
#pragma unroll
  for (int i = 0; i < kKeysPer; ++i) old[i] = j0 + tid + i * kJoin < j1 ? a.weights_in[(size_t)zh * c.C + j0 + tid + i * kJoin] : 0.f;
  wait_for_previous();
  const float* scores = p.scores + (size_t)zh * c.C * p.score_rows;
  float4 x[kKeysPer];  // those of the first 4 rows are on their way before the rows' maxima are known
#pragma unroll
  for (int i = 0; i < kKeysPer; ++i) {
    const int j = j0 + tid + i * kJoin;
    x[i] = j < min(j1, most) ? scores_of(scores + (size_t)j * p.score_rows, p.score_rows) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int row = warp; row < (p.rows + 3) / 4 * 4; row += kJoin / 32) {
    float mx = -INFINITY, l = 0.f;
    const int limit = tiles && row < p.rows ? sp.limit(a, row / a.rep) : 0;
    const bool seen = limit > 0;
    if (seen) {
      const int u = row / R, r = row % R;
      const long long first = before + ((long long)h * p.row_tiles + u) * cost;
      const int c0 = holder(first + kBegin), n = holder(first + cost - 1) - c0 + 1;
      if (n == 1) {
        const float2 s = p.stats[((size_t)zh * p.row_tiles + u) * R + r];
        mx = s.x, l = s.y;
      } else {
        for (int k = lane; k < n; k += 32) mx = fmaxf(mx, part_of(first, c0, c0 + k)[r]);
#pragma unroll
        for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
        for (int k = lane; k < n; k += 32) {
          const float* part = part_of(first, c0, c0 + k);
          l += part[R + r] * (part[r] == -INFINITY ? 1.f : ex2(part[r] - mx));
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
      }
    }
    if (lane == 0) sm[row] = mx == -INFINITY ? 0.f : mx, sinv[row] = seen ? 1.f / l : 0.f, seen_to[row] = limit;
  }
  __syncthreads();
  float add[kKeysPer] = {};
  for (int row = 0; row < p.rows; row += 4) {
    const float4 m = *reinterpret_cast<const float4*>(sm + row), w = *reinterpret_cast<const float4*>(sinv + row);
    const int4 to = *reinterpret_cast<const int4*>(seen_to + row);
#pragma unroll
    for (int i = 0; i < kKeysPer; ++i) {
      const int j = j0 + tid + i * kJoin;
      if (row && j < min(j1, most)) x[i] = scores_of(scores + (size_t)j * p.score_rows + row, p.score_rows);
    }
#pragma unroll
    for (int i = 0; i < kKeysPer; ++i) {
      const int j = j0 + tid + i * kJoin;
      if (j < to.x) add[i] += ex2(x[i].x - m.x) * w.x;
      if (j < to.y) add[i] += ex2(x[i].y - m.y) * w.y;
      if (j < to.z) add[i] += ex2(x[i].z - m.z) * w.z;
      if (j < to.w) add[i] += ex2(x[i].w - m.w) * w.w;
    }
  }
#pragma unroll
  for (int i = 0; i < kKeysPer; ++i) {
    const int j = j0 + tid + i * kJoin;
    if (j < j1) c.weight[(size_t)zh * c.C + j] = old[i] + add[i];
  }
}

// ------------------------------------------------------------------ host
struct RowsPlan {
  int nt, row_tiles, rows, score_rows;
  int zs, hs;  // sequences and heads of a launch: all, some sequences with all heads, or some heads of one
  long long parts, stats, scores;  // floats
};
// The scores that the weights are formed from take up to 192 bytes per position and head, more than
// what is stored of them, and go by the capacity (lengths are known on the device only). So a call
// takes sequences and heads in groups of so many bytes of scores, or one head at a time.  A group costs some
// 25 us of launches and up to 50 of idle SMs at its end: 48 rows over 256 heads of 131072 positions (6.4 GB in all)
// 10.5 ms without groups, 12.1 in groups of 256 MB, 10.9 of 1 GB; 0.20, 0.95 and 0.39 where only 300 are stored.
constexpr long long kScoreBytes = 1LL << 30;

static RowsPlan plan_rows(const Cache& c, int rep, int N, bool weights) {
  RowsPlan p;
  p.rows = rep * N;
  p.nt = p.rows <= 8 ? 1 : 2;
  p.row_tiles = (p.rows + 8 * p.nt - 1) / (8 * p.nt);
  p.score_rows = p.rows <= 2 ? 2 : (p.rows + 3) / 4 * 4;
  p.parts = 2LL * kGridMax * 8 * p.nt * (c.D + 2);
  const long long heads = std::max(1LL, kScoreBytes / (4LL * c.C * p.score_rows));  // of a group
  p.zs = weights ? (int)std::min<long long>(c.Z, std::max(1LL, heads / c.H)) : c.Z;
  p.hs = weights ? (int)std::min<long long>(c.H, heads) : c.H;
  p.stats = weights ? 2LL * p.zs * p.hs * p.row_tiles * 8 * p.nt : 0;
  p.scores = weights ? (long long)p.zs * p.hs * c.C * p.score_rows : 0;
  return p;
}

size_t rows_workspace(const qflash_kv4_cache* c, int Hq, int N, bool weights) {
  const RowsPlan p = plan_rows(view(c), Hq / c->H, N, weights);
  return (size_t)(p.parts + p.stats + p.scores) * 4;
}

template <int D, int NT, bool FP16>
static int launch_rows(RowsArgs r, int dev, cudaStream_t s) {
  const Cache& c = r.a.c;
  constexpr uint32_t smem = rows_smem<D, NT>();
  static std::atomic<int> per_sm_on[kDevices];  // 0: not asked yet
  std::atomic<int>& per_sm = per_sm_on[dev];
  if (!per_sm.load()) {
    int n = 0;
    if (cudaFuncSetAttribute(rows_kernel<D, NT, FP16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaFuncSetAttribute(rows_kernel<D, NT, FP16>, cudaFuncAttributePreferredSharedMemoryCarveout, 100) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rows_kernel<D, NT, FP16>, kWarps * 32, smem) != cudaSuccess || n < 1)
      return set_err(QFLASH_ERR_LAUNCH, "kv4 rows: occupancy: %s", cudaGetErrorString(cudaGetLastError()));
    per_sm.store(n);
  }
  const long long units = (long long)c.Z * c.H * r.row_tiles, tiles = (c.C + kTile - 1) / kTile;
  // Short caches: a unit to a CTA, since joining costs a kernel; with longer ones, or few units that have their
  // weights to add up, SMs would idle for too long.  One kernel and two, us at rep 4, bf16: 8 heads of 333 positions
  // of 64 5.4 and 8.2; head dim 128, 8 heads of 512 7.6 and 9.1, of 1024 11.2 and 9.1 (which the launch saved makes up
  // for), with weights 15.9 and 9.2; 128 heads of 1024 11.7 and 18.5, 512 heads 24.7 and 39.5; 8 heads of 2048 some
  // 17 and 10.3.
  r.single = (tiles <= (r.scores && units < 64 ? 4 : 8) || (units >= 256 && tiles <= 16)) && (!r.scores || r.row_tiles == 1);
  if (r.single) {
    r.grid = (int)units;
    rows_kernel<D, NT, FP16><<<r.grid, kWarps * 32, smem, s>>>(r);
    return check_launch("kv4 rows", r.grid);
  }
  r.grid = (int)std::min<long long>(std::min<long long>((long long)sm_count(dev) * per_sm.load(), kGridMax), units * tiles);
  rows_kernel<D, NT, FP16><<<r.grid, kWarps * 32, smem, s>>>(r);
  if (int rc = check_launch("kv4 rows", r.grid)) return rc;
  const unsigned grid = (unsigned)(c.Z * c.H) * (r.rows + (r.scores ? (c.C + kChunk - 1) / kChunk : 0));
  launch_behind(rows_finish_kernel<D, NT, FP16>, grid, kJoin, s, r);
  return check_launch("kv4 rows finish", grid);
}

static int launch_rows(const RowsArgs& r, int nt, bool fp16, int dev, cudaStream_t s) {
  if (r.a.c.D == 64)
    return nt == 1 ? (fp16 ? launch_rows<64, 1, true>(r, dev, s) : launch_rows<64, 1, false>(r, dev, s))
                   : (fp16 ? launch_rows<64, 2, true>(r, dev, s) : launch_rows<64, 2, false>(r, dev, s));
  return nt == 1 ? (fp16 ? launch_rows<128, 1, true>(r, dev, s) : launch_rows<128, 1, false>(r, dev, s))
                 : (fp16 ? launch_rows<128, 2, true>(r, dev, s) : launch_rows<128, 2, false>(r, dev, s));
}

// What of a call belongs to nz sequences from z on, and nh heads from h on (all heads, or one sequence).
static AttendArgs group_of(AttendArgs a, int z, int nz, int h, int nh) {
  const int64_t head = (int64_t)z * a.c.H + h, at = head * a.c.C;
  for (int i = 0; i < 2; ++i) a.c.codes[i] += at * (a.c.D / 2), a.c.param[i] += at;
  a.c.weight += at, a.c.lens += z;
  a.q = (const uint16_t*)a.q + z * a.qs[0] + (int64_t)h * a.rep * a.qs[1];
  a.out = (uint16_t*)a.out + z * a.os[0] + (int64_t)h * a.rep * a.os[1];
  if (a.new_lens) a.new_lens += z;
  if (a.weights_in) a.weights_in += at;
  a.c.Z = nz, a.c.H = nh;
  return a;
}

int attend_rows(const AttendArgs& a, bool fp16, void* ws, int dev, cudaStream_t s) {
  const bool weights = a.weights_in != nullptr;
  const RowsPlan p = plan_rows(a.c, a.rep, a.N, weights);
  RowsArgs r;
  r.rows = p.rows;
  r.row_tiles = p.row_tiles;
  r.score_rows = p.score_rows;
  r.magic_k = fp16 ? kMagicFp16 : kMagicBf16;
  r.magic_v = kMagicBf16;
  r.vec_q = (((uintptr_t)a.q | (a.qs[0] * 2) | (a.qs[1] * 2) | (a.qs[2] * 2)) & 15) == 0;
  r.parts = (float*)ws;
  r.stats = (float2*)(r.parts + p.parts);
  r.scores = weights ? r.parts + p.parts + p.stats : nullptr;
  for (int z = 0; z < a.c.Z; z += p.zs)
    for (int h = 0; h < a.c.H; h += p.hs) {
      r.a = group_of(a, z, std::min(p.zs, a.c.Z - z), h, std::min(p.hs, a.c.H - h));
      if (int rc = launch_rows(r, p.nt, fp16, dev, s)) return rc;
    }
  return QFLASH_OK;
}

}  // namespace kv4
}  // namespace qfb
