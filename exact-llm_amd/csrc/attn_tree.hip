// Attention of drafted token trees over the cache: the q/k/v epilogue, RoPE, qrow, scores, softmax and p.V of
// exact_llm.py:164-176 for rows of which each sees the cached positions and the nodes its mask names.
//
// A tree's nodes lie behind the cached positions, node i at base + i, while RoPE turns a node by its depth, so the key of an
// accepted node is right wherever it is moved to afterwards. Rows of padding nodes are computed as the others are, over all keys,
// and come out as zeros.
#include "exact_common.h"
#include "abi_util.h"
#include "sample_ops.h"
#include <type_traits>

namespace exact {

#define TREE_T 64            // nodes of a tree: one bit each of a mask
#define TREE_SMAX (1 << 20)
#define TREE_KG 64           // keys of a score group: d is kept against the group's own maximum
#define TREE_CK 128          // keys a block of k_tree_pv
// Positions up to which one launch follows the epilogue, twice as many from TREE_SHORT_ROWS (row, head)s on. us a layer in a graph, one
// launch and four: 28 heads over 4 of 128, 8 nodes at 40 / 200 / 440 / 600 positions 15.9 / 19.9 / 28.5 / 39.9 and 23.8 / 24.0 / 24.0 /
// 23.8, four trees of 32 at 40 / 200 / 440 18.9 / 22.7 / 31.5 and 35.1 / 39.1 / 47.0; 40 over 8, 32 nodes at 440 29.5 and 29.4, four trees
// 55 and 58, at 600 78 and 63; 14 over 2 of 64, 8 nodes at 40 / 240 / 440 13.2 / 15.7 / 22.5 and 21.4 / 21.5 / 21.6.
#define TREE_SHORT 256
#define TREE_SHORT_ROWS 1024
#define TREE_MT 5            // most 16-row tiles of a block of k_tree_pv

// a sequence of the call: its slot, first node position and the nodes that it has (bit j: node j is real and inside the cache)
struct TreeSeq {
  int64_t slot;
  int base, S;   // S: positions up to the last node
  uint64_t live;
};

struct TreeArgs {
  const int32_t *slot, *base, *depth, *nodes;
  const int64_t* mask;
  int nslots, B, T, H, KV, G, Smax, rope_n, keys;
  int M, MP, NG;   // rows of a (sequence, KV head): (node, head of the group); padded to whole tiles; score groups
  int64_t Sp;      // padded score row
};

// Workspace, for each (sequence, KV head) and row m = node G + head of the group
struct TreeWork {
  int8_t* qd;      // [MP][2][HD]: digits of the quantised query, x = 256 hi + lo + 128
  int32_t *shq, *qsum;   // [MP]: its shift and sum
  int64_t *cm, *es;      // [MP][NG] maximum score of a group; [MP] sum of exponentials
  uint64_t* acc;   // [MP][HD]: p.V
  int32_t* neg;    // [MP]: an exponential is negative (of an exp table with negative entries)
  TreeSeq* seq;    // of each sequence, as the first launch finds it
  uint32_t* d;     // [MP][Sp]: maximum of the group - score (at most EXP_FAR; EXP_UNSEEN), then p: of 128 keys' 512 bytes the first
                   // 384, of every 4 keys three dwords with one digit each; the exponentials if one is negative
};

// for whole waves
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& A, int b) {
  const int lane = threadIdx.x & 63;
  TreeSeq q;
  q.slot = A.slot[b];
  q.base = A.base[b];
  const int n = A.nodes ? A.nodes[b] : A.T;
  bool again = false;   // a sequence before it has this slot
  for (int j = lane; j < b; j += 64) again |= A.slot[j] == q.slot && (!A.nodes || A.nodes[j] > 0);
  bool ok = !__any(again) && q.slot >= 0 && q.slot < A.nslots && q.base >= 0 && q.base < A.keys && lane < A.T && lane < n &&
            q.base + lane < A.keys;
  if (ok) {
    const int64_t at = (int64_t)q.base + A.depth[(int64_t)b * A.T + lane];
    ok = at >= 0 && at < A.rope_n;
  }
  q.live = __ballot(ok);
  q.S = q.live ? q.base + 64 - __clzll((long long)q.live) : 0;
  return q;
}

// grid (B T, H + 2 KV), one wave a head: y = shr(t, 28 - s) + b, RoPE at base + depth, qrow; query digits to the workspace, key and
// value to the cache at base + node. Queries of dead nodes are zeros. Latency: 3.6 us for 8 rows of 18 heads of 64, 12.5 us for 256 rows of
// 56 heads of 128 (20 MB read and written; clear_t writes 15 more).
template <int HD>
__global__ __launch_bounds__(64) void k_tree_qkv(int64_t* __restrict__ t, const int32_t* __restrict__ s,
                                                 const int64_t* __restrict__ b, const int64_t* __restrict__ cos_t,
                                                 const int64_t* __restrict__ sin_t, int16_t* __restrict__ kq,
                                                 int32_t* __restrict__ sk, int64_t* __restrict__ v, TreeArgs A, TreeWork W,
                                                 int clear_t) {
  constexpr int KS = HD / 64;
  const int r = blockIdx.x, hs = blockIdx.y, lane = threadIdx.x, bt = r / A.T, node = r - bt * A.T;
  const int64_t N = (int64_t)(A.H + 2 * A.KV) * HD;
  int64_t* row = t + r * N + hs * HD;
  // the totals first: the sequence's facts take two loads in turn
  int64_t raw[KS], bias[KS], y[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    raw[i] = row[lane + 64 * i];
    bias[i] = b ? b[hs * HD + lane + 64 * i] : 0;
  }
  const int sh = 28 - s[r];
  const TreeSeq q = tree_seq(A, bt);
  if (node == 0 && hs == 0 && lane == 0) W.seq[bt] = q;
  const bool live = q.live >> node & 1;
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    y[i] = shr64(raw[i], sh) + bias[i];
    if (clear_t) row[lane + 64 * i] = 0;
  }
  if (!live && hs >= A.H) return;
  const int64_t at = (q.slot * A.KV + (hs - A.H) % A.KV) * A.Smax + q.base + node;   // of a key or value head
  if (hs >= A.H + A.KV) {
#pragma unroll
    for (int i = 0; i < KS; ++i) v[at * HD + lane + 64 * i] = y[i];
    return;
  }
  const int64_t p = live ? (int64_t)q.base + A.depth[r] : 0;
  int64_t z[KS], m = 0;
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int j = lane + 64 * i;
    int64_t rot;   // of (a, b): (-b, a)
    if constexpr (KS == 1) {
      rot = __shfl_xor((long long)y[0], 32, 64);
      rot = lane < 32 ? -rot : rot;
    } else {
      rot = i == 0 ? -y[1] : y[0];
    }
    z[i] = live ? shr64(y[i] * cos_t[p * HD + j] + rot * sin_t[p * HD + j], EXACT_F) : 0;
    m = max64(m, abs64(z[i]));
  }
  m = wave_max64(m);
  const int sv = max(bitlen64(m) - 15, 0);
  int x[KS], sum = 0;
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    const int64_t w = shr64(z[i], sv);
    x[i] = (int)(w > 32767 ? 32767 : (w < -32767 ? -32767 : w));
    sum += x[i];
  }
  if (hs >= A.H) {
#pragma unroll
    for (int i = 0; i < KS; ++i) kq[at * HD + lane + 64 * i] = (int16_t)x[i];
    if (lane == 0) sk[at] = sv;
    return;
  }
  const int kh = hs / A.G;
  const int64_t mrow = ((int64_t)bt * A.KV + kh) * A.MP + node * A.G + hs - kh * A.G;
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    W.qd[mrow * 2 * HD + lane + 64 * i] = (int8_t)(x[i] >> 8);
    W.qd[mrow * 2 * HD + HD + lane + 64 * i] = (int8_t)((x[i] & 255) - 128);
  }
  sum = (int)wave_sum64(sum);
  if (lane == 0) {
    W.shq[mrow] = sv;
    W.qsum[mrow] = sum;
  }
}

// grid (score groups x mparts, KV, B), 4 waves: the scores of 64 keys against all rows, 16 rows a tile, tiles dealt out to the waves of
// mparts blocks. On the matrix cores from int8 digits: q.k = 65536 HH + 256 (HL + LH) + LL + 128 (sum q + sum k) - 16384 HD (digit sums
// below 2^23), with the keys (split into digits once, in LDS) as the rows of v_mfma_i32_16x16x64_i8 and the query rows as its columns; the
// sums go into LL's accumulator. rs(q.k INV, 32 - sq - sk) is made in float64 where that is exact: shifts of -1 to 32 and INV below 2^14,
// so that |q.k INV| < 2^51, the scales are powers of two and floor(x + 1/2) the rounding half up; in int64 otherwise. 62 million scores of
// 128 dimensions (40 heads over 8, four trees of 64 at 6001 positions) take 100 us: 19 vector instructions a score keep the SIMDs 46% busy,
// the matrix cores 15%, and 248 MB of distances are written; 10.3 us for 28 heads over 4, a tree of 26 at 1793.
template <int HD>
__global__ __launch_bounds__(256, 4) void k_tree_scores(const int16_t* __restrict__ kq, const int32_t* __restrict__ sk, TreeArgs A,
                                                     TreeWork W, int INV, int mparts) {
  constexpr int KS = HD / 64, KT = TREE_KG / 16, UN = HD / 16;
  __shared__ __attribute__((aligned(16))) int8_t kd[2][TREE_KG][HD];
  __shared__ __attribute__((aligned(16))) int kterm[TREE_KG], ksh[TREE_KG];
  const int c = blockIdx.x / mparts, mp = blockIdx.x - c * mparts, kh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, qt = lane >> 4, k0 = c * TREE_KG;
  const TreeSeq q = W.seq[b];
  if (k0 >= q.S) return;   // uniform over the block
  const int64_t row0 = ((int64_t)b * A.KV + kh) * A.MP;
  int qlow = 0, qhigh = 0;   // of the rows' shifts, in flight with the keys
  for (int i = lane; i < A.M; i += 64) {
    const int sq = W.shq[row0 + i];
    qlow = min(qlow, sq);
    qhigh = max(qhigh, sq);
  }
  {   // four threads a key
    const int64_t cbase = (q.slot * A.KV + kh) * A.Smax;
    const int j = tid >> 2, key = min(k0 + j, q.S - 1);
    const v4i* kr = reinterpret_cast<const v4i*>(kq + (cbase + key) * HD);
    v4i raw[UN / 4][2];
#pragma unroll
    for (int i = 0; i < UN / 4; ++i) {   // 16 dimensions each
      raw[i][0] = kr[2 * ((tid & 3) + 4 * i)];
      raw[i][1] = kr[2 * ((tid & 3) + 4 * i) + 1];
    }
    const int sh = sk[cbase + key];
    int hs = 0, ls = 0;
#pragma unroll
    for (int i = 0; i < UN / 4; ++i) {
      v4i hi, lo;
      split_digits(raw[i][0], raw[i][1], hi, lo);
      const int at = 16 * (((tid & 3) + 4 * i) ^ (j >> 1 & (UN - 1)));   // no two keys of a read on the same banks
      *reinterpret_cast<v4i*>(&kd[0][j][at]) = hi;
      *reinterpret_cast<v4i*>(&kd[1][j][at]) = lo;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        hs = __builtin_amdgcn_sdot4(hi[w], 0x01010101, hs, false);
        ls = __builtin_amdgcn_sdot4(lo[w], 0x01010101, ls, false);
      }
    }
    int t = 256 * hs + ls;
    t += dpp32<0xB1>(t);
    t += dpp32<0x4E>(t);
    if ((tid & 3) == 0) {
      kterm[j] = 128 * (t + 128 * HD) - 16384 * HD;   // 128 sum k less its constant: |.| < 2^30
      ksh[j] = sh;
    }
  }
  __syncthreads();
  const int smax = wave_max_i32(ksh[lane]), smin = ~wave_max_i32(~ksh[lane]);
  const int kx = col >> 1 & (UN - 1);
  // MODE 0: float64, every key is seen by every row; 1: float64, 2: int64, keys by the lane's bits (4 kt + i)
  auto tiles = [&](auto mode) {
    constexpr int MODE = decltype(mode)::value;
    constexpr bool F = MODE < 2;
    typedef std::conditional_t<F, double, int64_t> X;
    for (int m0 = 16 * (mp * 4 + wave); m0 < A.M; m0 += 64 * mparts) {
      asm volatile("" ::: "memory");   // the keys' digits are read from LDS for every tile: held in registers they cost half the waves
      const int m = min(m0 + col, A.M - 1);
      const int8_t* qr = W.qd + (row0 + m) * 2 * HD + 16 * qt;
      v4i qh[KS], ql[KS];
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        qh[i] = *reinterpret_cast<const v4i*>(qr + 64 * i);
        ql[i] = *reinterpret_cast<const v4i*>(qr + HD + 64 * i);
      }
      const int sq = W.shq[row0 + m], qterm = 128 * W.qsum[row0 + m];   // < 2^29
      uint32_t sees = 0;
      if constexpr (MODE > 0) {
        const int node = m / A.G;
        const bool live = q.live >> node & 1;
        const uint64_t seen = live ? (uint64_t)A.mask[(int64_t)b * A.T + node] & q.live : 0;
        const int upto = live ? q.base : 0;   // keys below it are seen
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int si = k0 + 16 * kt + 4 * qt + i;
            const bool ok = si < upto || (si >= q.base && si < q.S && (seen >> ((si - q.base) & 63) & 1));
            sees |= (uint32_t)ok << (4 * kt + i);
          }
      }
      X x[KT][4], mx = F ? (X)-__builtin_inf() : (X)INT64_MIN;
      const double qs = (double)INV * __builtin_ldexp(1.0, F ? sq - 32 : 0);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        v4i hh = v4i{}, mid = v4i{}, ll = *reinterpret_cast<const v4i*>(&kterm[16 * kt + 4 * qt]);
        const v4i sh = *reinterpret_cast<const v4i*>(&ksh[16 * kt + 4 * qt]);
#pragma unroll
        for (int i = 0; i < 4; ++i) ll[i] += qterm;
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          const v4i hi = *reinterpret_cast<const v4i*>(&kd[0][16 * kt + col][16 * ((4 * i + qt) ^ kx)]);
          const v4i lo = *reinterpret_cast<const v4i*>(&kd[1][16 * kt + col][16 * ((4 * i + qt) ^ kx)]);
          hh = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, qh[i], hh, 0, 0, 0);
          mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi, ql[i], mid, 0, 0, 0);
          ll = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, ql[i], ll, 0, 0, 0);
          mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo, qh[i], mid, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (F) {
            const double dot = __builtin_fma((double)(256 * hh[i] + mid[i]), 256.0, (double)ll[i]);   // the first below 2^30
            x[kt][i] = __builtin_floor(__builtin_fma(dot, __builtin_ldexp(qs, sh[i]), 0.5));   // exact before and after the half
            if (MODE == 0 || (sees >> (4 * kt + i) & 1)) mx = __builtin_fmax(mx, x[kt][i]);
          } else {
            const int64_t dot = ((int64_t)hh[i] << 16) + ((int64_t)mid[i] << 8) + ll[i];
            x[kt][i] = shr64(dot * INV, 32 - sq - sh[i]);
            if (sees >> (4 * kt + i) & 1) mx = max64(mx, x[kt][i]);
          }
        }
      }
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) {
        if constexpr (F) mx = __builtin_fmax(mx, __shfl_xor(mx, o));
        else mx = max64(mx, (int64_t)__shfl_xor((long long)mx, o));
      }
      if (m0 + col >= A.M) continue;
      uint32_t* dr = W.d + (row0 + m) * A.Sp + k0 + 4 * qt;
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        v4i dv;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (F) {
            dv[i] = (int)(uint32_t)__builtin_fmin(mx - x[kt][i], (double)EXP_FAR);
          } else {
            const uint64_t gap = (uint64_t)mx - (uint64_t)x[kt][i];
            dv[i] = (int)(gap < EXP_FAR ? (uint32_t)gap : EXP_FAR);
          }
          if (MODE > 0 && !(sees >> (4 * kt + i) & 1)) dv[i] = EXP_UNSEEN;
        }
        *reinterpret_cast<v4i*>(dr + 16 * kt) = dv;
      }
      if (qt == 0) {
        int64_t w;
        if constexpr (F) w = mx == -__builtin_inf() ? INT64_MIN : (int64_t)mx;
        else w = mx;
        W.cm[(row0 + m) * A.NG + c] = w;
      }
    }
  };
  const uint64_t dead = ~q.live & (A.T < 64 ? (1ULL << A.T) - 1 : ~0ULL);
  const bool f64 = smin >= 0 && smax <= 33 && INV > 0 && INV < (1 << 14) && !__any(qlow < 0 || qhigh > 33 || qhigh + smax > 33);
  if (!f64) tiles(std::integral_constant<int, 2>{});
  else if (k0 + TREE_KG <= q.base && dead == 0) tiles(std::integral_constant<int, 0>{});
  else tiles(std::integral_constant<int, 1>{});
}

// the four bytes of a[0 .. 3] as four dwords, one of each byte, with the sign bits turned: of numbers with 128 added to every byte
// these are their balanced base-256 digits
__device__ __forceinline__ void byte_planes(const uint32_t* a, int& b0, int& b1, int& b2, int& b3) {
  const uint32_t x = __builtin_amdgcn_perm(a[1], a[0], 0x05010400u), y = __builtin_amdgcn_perm(a[3], a[2], 0x05010400u);
  const uint32_t z = __builtin_amdgcn_perm(a[1], a[0], 0x07030602u), w = __builtin_amdgcn_perm(a[3], a[2], 0x07030602u);
  b0 = (int)(__builtin_amdgcn_perm(y, x, 0x05040100u) ^ 0x80808080u);
  b1 = (int)(__builtin_amdgcn_perm(y, x, 0x07060302u) ^ 0x80808080u);
  b2 = (int)(__builtin_amdgcn_perm(w, z, 0x05040100u) ^ 0x80808080u);
  b3 = (int)(__builtin_amdgcn_perm(w, z, 0x07060302u) ^ 0x80808080u);
}

// grid (M, KV, B), one block a row: its maximum from the groups', the exponentials, their sum, and p as its three balanced base-256
// digits over the distances (p is made as prob20 makes it, whose conditions hold where no exponential is negative); clears the p.V
// totals. The first distances are in flight while the maximum is found and their exponentials stay in registers; those of longer rows
// are made again. A quad of keys lies within the lane's own 128 keys, which one wave reads before it writes them. Bound by about 40
// vector instructions a distance, which keep the SIMDs 73% busy: 105 us for 62 million distances, 7 bytes read and written each (4.1 TB/s;
// with distances and digits in 24 bits, a quarter less, the launch took 95 and the value product as much more). Seven waves a SIMD are
// asked for, because with all the registers every table entry of the row is loaded ahead and few waves are left (332 us).
template <int HD>
__global__ __launch_bounds__(256, 7) void k_tree_exp(const int32_t* __restrict__ expt, TreeArgs A, TreeWork W) {
  __shared__ int64_t red[2][16];
  __shared__ int anyneg;
  constexpr int PF = 6;
  const int tid = threadIdx.x;
  const int b = A.B - 1 - blockIdx.z, kh = A.KV - 1 - blockIdx.y;   // last written first: what the caches still hold
  const TreeSeq q = W.seq[b];
  const int64_t row = ((int64_t)b * A.KV + kh) * A.MP + blockIdx.x;
  for (int i = tid; i < HD; i += 256) W.acc[row * HD + i] = 0;
  if (tid == 0) anyneg = 0;
  const int ng = (q.S + TREE_KG - 1) / TREE_KG, n = ng * TREE_KG;
  const int64_t* cm = W.cm + row * A.NG;
  uint32_t* d = W.d + row * A.Sp;
  v4i pre[PF];
  int64_t top[PF], mx = INT64_MIN;
#pragma unroll
  for (int k = 0; k < PF; ++k)
    if (4 * tid + 1024 * k < n) {
      pre[k] = *reinterpret_cast<const v4i*>(d + 4 * tid + 1024 * k);
      top[k] = cm[(4 * tid + 1024 * k) / TREE_KG];
    }
  for (int i = tid; i < ng; i += 256) mx = max64(mx, cm[i]);
  mx = block_max64_1(mx, red[0]);
  int64_t es = 0;
  bool neg = false;
  auto exps = [&](v4i x, int64_t t) {
    const uint32_t gap = exp_gap(mx, t);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = lut_exp_kept(expt, gap, (uint32_t)x[j]);
    return x;
  };
  auto add = [&](v4i x) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      es += x[j];
      neg |= x[j] < 0;
    }
  };
#pragma unroll
  for (int k = 0; k < PF; ++k)
    if (4 * tid + 1024 * k < n) add(pre[k] = exps(pre[k], top[k]));
  for (int i = 4 * tid + 1024 * PF; i < n; i += 1024) add(exps(*reinterpret_cast<const v4i*>(d + i), cm[i / TREE_KG]));
  if (neg) anyneg = 1;
  es = block_sum64_1(es, red[1]);
  neg = anyneg;
  if (tid == 0) {
    W.es[row] = es;
    W.neg[row] = neg;
  }
  const double es20 = sum20(es), rb = sum20_rcp(es20);   // of a row that sees nothing: every e is 0
  auto put = [&](int i, v4i e) {
    if (neg) {
      *reinterpret_cast<v4i*>(d + i) = e;
      return;
    }
    uint32_t x[4], *o = d + (i & -128) + 3 * ((i & 127) >> 2);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const double ef = (double)(uint32_t)e[j], p = __builtin_floor(ef * rb);
      x[j] = (uint32_t)p + 0x808080u + (__builtin_fma(-p, es20, ef) >= es20);
    }
    int b0, b1, b2, b3;
    byte_planes(x, b0, b1, b2, b3);
    o[0] = b0, o[1] = b1, o[2] = b2;
  };
#pragma unroll
  for (int k = 0; k < PF; ++k)
    if (4 * tid + 1024 * k < n) put(4 * tid + 1024 * k, pre[k]);
  for (int i = 4 * tid + 1024 * PF; i < n; i += 1024) put(i, exps(*reinterpret_cast<const v4i*>(d + i), cm[i / TREE_KG]));
}

// grid (KV B, row groups, ksplit), 8 waves: p.V of MT 16-row tiles over a run of the keys, added to the rows' totals (64-bit atomics, exact
// in any order). 128 keys a step: every thread brings the digits of p of 4 keys of MT rows, which go through LDS to the matrix cores. A
// wave takes 16 dimensions of the step's keys (hd 64: of half of them), splits its values into digits in registers and holds the products'
// sums of all the rows. p (0 .. 2^20) and v (below 2^23) have three balanced base-256 digits each; where a wave's values have more, the
// upper five digits' products go to the totals by themselves. The products of one weight sum up in int32 (keys x 3 pairs x 2^14: below 2^31
// for 32768 keys a block) and are joined modulo 2^64 at the end. The row groups of a run of keys lie next to each other on one XCD, whose
// L2 gives them the values that the first of them reads. 120 us at the 62 million weights (five tiles a block), the matrix cores 27% and
// the vector units 25% busy: the sums of five tiles leave registers for two waves a SIMD, which wait half of their time. 12.5 us for 28
// heads over 4, a tree of 26 at 1793.
template <int HD, int MT>
__global__ __launch_bounds__(512) void k_tree_pv(const int64_t* __restrict__ v, TreeArgs A, TreeWork W) {
  constexpr int NS = TREE_CK * HD / 8192, NC = 5, ROWS = 16 * MT;   // a wave's 64-key parts of a step; weights
  __shared__ __attribute__((aligned(16))) int8_t pd[2][3][ROWS][TREE_CK];
  const int kh = blockIdx.x % A.KV, b = blockIdx.x / A.KV, mg = blockIdx.y * ROWS, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, qt = lane >> 4;
  const TreeSeq q = W.seq[b];
  const int nch = (q.S + TREE_CK - 1) / TREE_CK, per = (nch + gridDim.z - 1) / gridDim.z;
  const int c0 = blockIdx.z * per, c1 = min(c0 + per, nch);
  if (c0 >= c1) return;
  const int64_t cbase = (q.slot * A.KV + kh) * A.Smax, row0 = ((int64_t)b * A.KV + kh) * A.MP;
  int neg = 0;
  for (int i = lane; i < min(ROWS, A.M - mg); i += 64) neg |= W.neg[row0 + mg + i];
  if (__any(neg)) {   // p of any size: 64-bit products
    for (int i = tid; i < ROWS * HD; i += 512) {
      const int m = mg + i / HD, dim = i % HD;
      if (m >= A.M) break;
      const bool whole = W.neg[row0 + m];
      const int64_t es = W.es[row0 + m];
      const uint32_t* d = W.d + (row0 + m) * A.Sp;
      uint64_t a = 0;
      for (int k = c0 * TREE_CK; k < min(c1 * TREE_CK, q.S); ++k) {
        const int8_t* x = reinterpret_cast<const int8_t*>(d + (k & -128) + 3 * ((k & 127) >> 2)) + (k & 3);
        const int64_t p = whole ? floordiv_pos(shl64((int32_t)d[k], 20), es) : 65536 * x[8] + 256 * x[4] + x[0];
        a += (uint64_t)p * (uint64_t)v[(cbase + k) * HD + dim];
      }
      atomicAdd(reinterpret_cast<unsigned long long*>(W.acc + (row0 + m) * HD + dim), (unsigned long long)a);
    }
    return;
  }
  const int slice = wave % (HD / 16), s0 = wave / (HD / 16);
  // the KV head's rows up to the last node, as a buffer: loads past them give 0 (S rows of at most 1 KiB: 2^30 bytes)
  const __amdgpu_buffer_rsrc_t vr =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<int64_t*>(v + cbase * HD), 0, q.S * (8 * HD), 0x00020000);
  const uint32_t vo = 8 * (16 * slice + col) + 16 * qt * (8 * HD);
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  v2u raw[16];
  auto load_v = [&](int k) {   // the lane's 16 keys of the 64 from k on
#pragma unroll
    for (int j = 0; j < 16; ++j) raw[j] = __builtin_amdgcn_raw_buffer_load_b64(vr, vo + (uint32_t)(k + j) * (8 * HD), 0, 0);
  };
  auto value = [&](int j) { return (uint64_t)raw[j][1] << 32 | raw[j][0]; };
  const int written = (q.S + TREE_KG - 1) / TREE_KG * TREE_KG;   // of the digits
  const int pr = tid >> 5, u = tid & 31;   // rows pr + 16 i, keys 4 u .. 4 u + 3 of a step
  uint32_t pp[MT][3];
  auto load_p = [&](int k) {
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = mg + pr + 16 * i;
      const bool in = m < A.M && k + 4 * u < written;
      const uint32_t* x = W.d + (row0 + m) * A.Sp + k + 3 * u;
#pragma unroll
      for (int a = 0; a < 3; ++a) pp[i][a] = in ? x[a] : 0;
    }
  };
  v4i acc[MT][NC];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[mt][i] = v4i{};
  auto put_p = [&](int8_t (*ps)[ROWS][TREE_CK]) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int a = 0; a < 3; ++a)
        *reinterpret_cast<uint32_t*>(&ps[a][pr + 16 * i][16 * ((u >> 2) ^ (pr >> 1 & 7)) + 4 * (u & 3)]) = pp[i][a];
  };
  load_p(c0 * TREE_CK);
  load_v(c0 * TREE_CK + 64 * s0);
  put_p(pd[0]);
  if (c0 + 1 < c1) load_p((c0 + 1) * TREE_CK);
  __syncthreads();
  for (int c = c0, n = 0; c < c1; ++c, n ^= 1) {
    const int k0 = c * TREE_CK;
    int8_t (*ps)[ROWS][TREE_CK] = pd[n];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int unit = 16 * ((4 * (s0 + s) + qt) ^ (col >> 1 & 7));   // no two rows of a read on the same banks
      v4i vd[3];
      uint32_t over = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t w = value(4 * i + j) + 0x808080ULL;   // in 24 bits if three digits hold it
          x[j] = (uint32_t)w;
          over |= (uint32_t)(w >> 32) | (x[j] & 0xff000000u);
        }
        int d[4];
        byte_planes(x, d[0], d[1], d[2], d[3]);
        vd[0][i] = d[0], vd[1][i] = d[1], vd[2][i] = d[2];
      }
      if (__any(over != 0)) {   // the upper digits' products, straight to the totals
#pragma unroll 1
        for (int k = 3; k < 8; ++k) {
          v4i vh;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t y = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              y |= (uint32_t)((value(4 * i + j) + 0x8080808080808080ULL) >> (8 * k) & 255) << (8 * j);
            vh[i] = (int)(y ^ 0x80808080u);
          }
#pragma unroll 1
          for (int mt = 0; mt < MT && mg + 16 * mt < A.M; ++mt)
#pragma unroll 1
            for (int a = 0; a < 3 && a + k < 8; ++a) {
              const v4i pa = *reinterpret_cast<const v4i*>(&ps[a][16 * mt + col][unit]);
              const v4i t = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa, vh, v4i{}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int m = mg + 16 * mt + 4 * qt + i;
                if (m < A.M)
                  atomicAdd(reinterpret_cast<unsigned long long*>(W.acc + (row0 + m) * HD + 16 * slice + col),
                            (unsigned long long)(long long)t[i] << (8 * (a + k)));
              }
            }
        }
      }
      // the next part's values, in flight during the products
      if (s + 1 < NS) load_v(k0 + 64 * (s0 + s + 1));
      else if (c + 1 < c1) load_v(k0 + TREE_CK + 64 * s0);
      __builtin_amdgcn_s_setprio(1);   // the SIMD's other wave splits values meanwhile: 317 us, 321 without
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int a = 0; a < 3; ++a) {
          const v4i pa = *reinterpret_cast<const v4i*>(&ps[a][16 * mt + col][unit]);
#pragma unroll
          for (int i = 0; i < 3; ++i) acc[mt][a + i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa, vd[i], acc[mt][a + i], 0, 0, 0);
        }
      __builtin_amdgcn_s_setprio(0);
    }
    if (c + 1 < c1) put_p(pd[n ^ 1]);
    if (c + 2 < c1) load_p(k0 + 2 * TREE_CK);
    __syncthreads();   // the buffer written now was read before the last one
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint64_t tot = 0;
#pragma unroll
      for (int k = 0; k < NC; ++k) tot += (uint64_t)(int64_t)acc[mt][k][i] << (8 * k);
      const int m = mg + 16 * mt + 4 * qt + i;
      if (m < A.M)
        atomicAdd(reinterpret_cast<unsigned long long*>(W.acc + (row0 + m) * HD + 16 * slice + col), (unsigned long long)tot);
    }
}

// Calls of at most 256 NGW positions, all of the layer after the epilogue in one launch: grid (KV B, row tiles), 8 waves. Wave w
// takes the 64-key groups w / 2 + 4 n (n < NGW) and, of p.V, half w % 2 of the dimensions; both halves make the same scores, whose
// distances stay in registers while the waves exchange the rows' maxima and sums, and p leaves the scores in the order in which
// the matrix cores take it (k slot 16 qt + 4 kt + i: key 16 kt + 4 qt + i), so that no key, p or value goes through LDS. Keys and
// values are read for every 16 rows, which bounds it from below; over few keys the four launches it replaces cost more. 9.5 us for 14
// heads over 2 of 64, 8 nodes at 37 positions: the chain of its loads and two barriers.
template <int HD, int NGW>
__global__ __launch_bounds__(512) void k_tree_short(const int16_t* __restrict__ kq, const int32_t* __restrict__ sk,
                                                    const int64_t* __restrict__ v, const int32_t* __restrict__ expt, TreeArgs A,
                                                    TreeWork W, int INV, int64_t* __restrict__ out, int32_t* __restrict__ obits) {
  constexpr int KS = HD / 64, SL = HD / 32, NC = 5, DPT = HD / 32;
  __shared__ uint64_t tot[16][HD];
  __shared__ int64_t xm[4][16], xs[4][16], ps[512];
  const int kh = blockIdx.x % A.KV, b = blockIdx.x / A.KV, m0 = 16 * blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave >> 1, half = wave & 1, col = lane & 15, qt = lane >> 4;
  const TreeSeq q = W.seq[b];
  const int64_t cbase = (q.slot * A.KV + kh) * A.Smax, row0 = ((int64_t)b * A.KV + kh) * A.MP;
  for (int i = tid; i < 16 * HD; i += 512) (&tot[0][0])[i] = 0;
  const int m = min(m0 + col, A.M - 1), node = m / A.G;
  const int8_t* qr = W.qd + (row0 + m) * 2 * HD + 16 * qt;
  v4i qh[KS], ql[KS];
#pragma unroll
  for (int i = 0; i < KS; ++i) {
    qh[i] = *reinterpret_cast<const v4i*>(qr + 64 * i);
    ql[i] = *reinterpret_cast<const v4i*>(qr + HD + 64 * i);
  }
  const int sq = W.shq[row0 + m], qterm = 128 * W.qsum[row0 + m];
  const bool live = q.live >> node & 1;
  const uint64_t seen = live ? (uint64_t)A.mask[(int64_t)b * A.T + node] & q.live : 0;
  const int upto = live ? q.base : 0, qmax = wave_max_i32(sq), qmin = ~wave_max_i32(~sq);
  const v4i ones = {0x01010101, 0x01010101, 0x01010101, 0x01010101};
  int64_t cm[NGW], mx = INT64_MIN;
  uint32_t d[NGW][4][4];
#pragma unroll
  for (int n = 0; n < NGW; ++n) {
    const int k0 = TREE_KG * (kw + 4 * n);
    cm[n] = INT64_MIN;
#pragma unroll
    for (int i = 0; i < 16; ++i) d[n][i / 4][i % 4] = EXP_UNSEEN;
    if (k0 >= q.S) continue;   // uniform over the wave
    v4i hi[4][KS], lo[4][KS], kterm[4], ksh[4];
    int smax = INT32_MIN, smin = INT32_MAX;
    uint32_t sees = 0;
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      const v4i* kr = reinterpret_cast<const v4i*>(kq + (cbase + min(k0 + 16 * kt + col, q.S - 1)) * HD + 16 * qt);
#pragma unroll
      for (int i = 0; i < KS; ++i) hi[kt][i] = kr[8 * i], lo[kt][i] = kr[8 * i + 1];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int si = k0 + 16 * kt + 4 * qt + i;
        ksh[kt][i] = sk[cbase + min(si, q.S - 1)];
        const bool ok = si < upto || (si >= q.base && si < q.S && (seen >> ((si - q.base) & 63) & 1));
        sees |= (uint32_t)ok << (4 * kt + i);
      }
    }
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      v4i h1 = v4i{}, l1 = v4i{};
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const v4i a = hi[kt][i], c = lo[kt][i];
        split_digits(a, c, hi[kt][i], lo[kt][i]);
        h1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi[kt][i], ones, h1, 0, 0, 0);
        l1 = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo[kt][i], ones, l1, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kterm[kt][i] = 128 * (256 * h1[i] + l1[i] + 128 * HD) - 16384 * HD + qterm;
        smax = max(smax, ksh[kt][i]);
        smin = min(smin, ksh[kt][i]);
      }
    }
    smax = wave_max_i32(smax);
    smin = ~wave_max_i32(~smin);
    const bool f64 = smin >= 0 && smax <= 33 && qmin >= 0 && qmax <= 33 && smax + qmax <= 33 && INV > 0 && INV < (1 << 14);
    auto scores = [&](auto fast) {   // as k_tree_scores
      constexpr bool F = decltype(fast)::value;
      typedef std::conditional_t<F, double, int64_t> X;
      X x[4][4], top = F ? (X)-__builtin_inf() : (X)INT64_MIN;
      const double qs = (double)INV * __builtin_ldexp(1.0, F ? sq - 32 : 0);
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        v4i hh = v4i{}, mid = v4i{}, ll = kterm[kt];
#pragma unroll
        for (int i = 0; i < KS; ++i) {
          hh = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi[kt][i], qh[i], hh, 0, 0, 0);
          mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(hi[kt][i], ql[i], mid, 0, 0, 0);
          ll = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo[kt][i], ql[i], ll, 0, 0, 0);
          mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(lo[kt][i], qh[i], mid, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (F) {
            const double dot = __builtin_fma((double)(256 * hh[i] + mid[i]), 256.0, (double)ll[i]);
            x[kt][i] = __builtin_floor(__builtin_ldexp(dot * qs, ksh[kt][i]) + 0.5);
          } else {
            x[kt][i] = shr64((((int64_t)hh[i] << 16) + ((int64_t)mid[i] << 8) + ll[i]) * INV, 32 - sq - ksh[kt][i]);
          }
          if (sees >> (4 * kt + i) & 1) top = x[kt][i] > top ? x[kt][i] : top;
        }
      }
#pragma unroll
      for (int o = 16; o < 64; o <<= 1) {
        X y;
        if constexpr (F) y = __shfl_xor(top, o);
        else y = (int64_t)__shfl_xor((long long)top, o);
        top = y > top ? y : top;
      }
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t gap;
          if constexpr (F) gap = (uint32_t)__builtin_fmin(top - x[kt][i], (double)EXP_FAR);
          else gap = (uint64_t)top - (uint64_t)x[kt][i] < EXP_FAR ? (uint32_t)((uint64_t)top - (uint64_t)x[kt][i]) : EXP_FAR;
          d[n][kt][i] = sees >> (4 * kt + i) & 1 ? gap : EXP_UNSEEN;
        }
      if constexpr (F) cm[n] = top == -__builtin_inf() ? INT64_MIN : (int64_t)top;
      else cm[n] = top;
    };
    if (f64) scores(std::true_type{});
    else scores(std::false_type{});
    mx = max64(mx, cm[n]);
  }
  // the first values, in flight during the softmax: the KV head's rows up to the last node as a buffer, loads past them give 0
  const __amdgpu_buffer_rsrc_t vr =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<int64_t*>(v + cbase * HD), 0, q.S * (8 * HD), 0x00020000);
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  v2u raw[2][16];
  auto load = [&](int it, v2u (&r)[16]) {   // group it % NGW of dimension block it / NGW
    const uint32_t o = 8 * (16 * (half * SL + it / NGW) + col) + (uint32_t)(TREE_KG * (kw + 4 * (it % NGW)) + 4 * qt) * (8 * HD);
#pragma unroll
    for (int j = 0; j < 16; ++j)
      r[j] = __builtin_amdgcn_raw_buffer_load_b64(vr, o + (16 * (j >> 2) + (j & 3)) * (8 * HD), 0, 0);
  };
  load(0, raw[0]);
  if (half == 0 && qt == 0) xm[kw][col] = mx;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) mx = max64(mx, xm[i][col]);
  int64_t es = 0;
  bool neg = false;
#pragma unroll
  for (int n = 0; n < NGW; ++n) {
    const uint32_t gap = exp_gap(mx, cm[n]);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = lut_exp_kept(expt, gap, d[n][kt][i]);
        es += e;
        neg |= e < 0;
        d[n][kt][i] = (uint32_t)e;
      }
  }
  es += (int64_t)__shfl_xor((long long)es, 16);
  es += (int64_t)__shfl_xor((long long)es, 32);
  if (half == 0 && qt == 0) xs[kw][col] = es;
  neg = __syncthreads_or(neg);
  es = xs[0][col] + xs[1][col] + xs[2][col] + xs[3][col];
  if (!neg) {
    const double es20 = sum20(es), rb = sum20_rcp(es20);
    v4i pd[NGW][3];
#pragma unroll
    for (int n = 0; n < NGW; ++n)
#pragma unroll
      for (int kt = 0; kt < 4; ++kt) {
        uint32_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // as prob20
          const double ef = (double)d[n][kt][i], p = __builtin_floor(ef * rb);
          x[i] = (uint32_t)p + 0x808080u + (__builtin_fma(-p, es20, ef) >= es20);
        }
        int b0, b1, b2, b3;
        byte_planes(x, b0, b1, b2, b3);
        pd[n][0][kt] = b0, pd[n][1][kt] = b1, pd[n][2][kt] = b2;
      }
    v4i acc[NC];
    uint64_t upper[4];
#pragma unroll
    for (int it = 0; it < SL * NGW; ++it) {
      const int n = it % NGW;
      if (n == 0) {
#pragma unroll
        for (int i = 0; i < NC; ++i) acc[i] = v4i{};
#pragma unroll
        for (int i = 0; i < 4; ++i) upper[i] = 0;
      }
      if (it + 1 < SL * NGW) load(it + 1, raw[(it + 1) & 1]);
      v2u (&r)[16] = raw[it & 1];
      if (TREE_KG * (kw + 4 * n) < q.S) {   // uniform over the wave
        v4i vd[3];
        uint32_t over = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t w = ((uint64_t)r[4 * i + j][1] << 32 | r[4 * i + j][0]) + 0x808080ULL;   // in 24 bits if three digits hold it
            x[j] = (uint32_t)w;
            over |= (uint32_t)(w >> 32) | (x[j] & 0xff000000u);
          }
          int b0, b1, b2, b3;
          byte_planes(x, b0, b1, b2, b3);
          vd[0][i] = b0, vd[1][i] = b1, vd[2][i] = b2;
        }
#pragma unroll
        for (int a = 0; a < 3; ++a)
#pragma unroll
          for (int i = 0; i < 3; ++i) acc[a + i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pd[n][a], vd[i], acc[a + i], 0, 0, 0);
        if (__any(over != 0)) {   // the other five digits
#pragma unroll 1
          for (int c = 3; c < 8; ++c) {
            v4i vh = v4i{};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const uint64_t w = ((uint64_t)r[j][1] << 32 | r[j][0]) + 0x8080808080808080ULL;
              vh[j / 4] |= (int)((uint32_t)(w >> (8 * c) & 255) << (8 * (j & 3)));
            }
            vh ^= (int)0x80808080;
#pragma unroll
            for (int a = 0; a < 3; ++a) {
              const v4i t = __builtin_amdgcn_mfma_i32_16x16x64_i8(pd[n][a], vh, v4i{}, 0, 0, 0);
#pragma unroll
              for (int i = 0; i < 4; ++i) upper[i] += (uint64_t)shl64(t[i], 8 * (a + c));
            }
          }
        }
      }
      if (n == NGW - 1) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint64_t t = upper[i];
#pragma unroll
          for (int k = 0; k < NC; ++k) t += (uint64_t)(int64_t)acc[k][i] << (8 * k);
          atomicAdd(reinterpret_cast<unsigned long long*>(&tot[4 * qt + i][16 * (half * SL + it / NGW) + col]), (unsigned long long)t);
        }
      }
    }
  } else {   // p of any size (an exp table with negative entries): 64-bit products, row by row
    if (wave == 0 && qt == 0) {
      xm[0][col] = mx;
      xs[0][col] = es;
    }
    for (int r = 0; r < 16 && m0 + r < A.M; ++r) {
      const int nr = (m0 + r) / A.G;
      const uint64_t sr = q.live >> nr & 1 ? (uint64_t)A.mask[(int64_t)b * A.T + nr] & q.live : 0;
      const int8_t* qp = W.qd + (row0 + m0 + r) * 2 * HD;
      uint64_t t = 0;
      for (int k0 = 0; k0 < q.S; k0 += 512) {
        const int k = k0 + tid;
        int64_t p = 0;
        __syncthreads();
        if (k < q.S && (k < q.base ? (bool)(q.live >> nr & 1) : (bool)(sr >> (k - q.base) & 1))) {
          int64_t dot = 0;
          for (int j = 0; j < HD; ++j) dot += (256 * qp[j] + qp[HD + j] + 128) * (int)kq[(cbase + k) * HD + j];
          const int64_t x = shr64(dot * INV, 32 - W.shq[row0 + m0 + r] - sk[cbase + k]);
          p = floordiv_pos(shl64(lut_exp(expt, xm[0][r], x), 20), xs[0][r]);
        }
        ps[tid] = p;
        __syncthreads();
        if (tid < HD)
          for (int i = 0; i < min(512, q.S - k0); ++i) t += (uint64_t)ps[i] * (uint64_t)v[(cbase + k0 + i) * HD + tid];
      }
      if (tid < HD) tot[r][tid] = t;
    }
  }
  __syncthreads();
  // 32 threads a row: out = shr(p.V, 20) and the head's bit length
  const int r = tid >> 5, l = tid & 31, mr = m0 + r;
  if (mr >= A.M) return;
  const int64_t o = ((int64_t)b * A.T + mr / A.G) * A.H + kh * A.G + mr % A.G;
  int bits = 0;
#pragma unroll
  for (int i = 0; i < DPT; ++i) {
    const int64_t x = shr64((int64_t)tot[r][l + 32 * i], 20);
    out[o * HD + l + 32 * i] = x;
    bits = max(bits, bitlen64(abs64(x)));
  }
  if (!obits) return;
  bits = max(bits, dpp32<0xB1>(bits));
  bits = max(bits, dpp32<0x4E>(bits));
  bits = max(bits, dpp32<0x141>(bits));
  bits = max(bits, dpp32<0x140>(bits));
  bits = max(bits, __shfl_xor(bits, 16));
  if (l == 0) obits[o] = bits;
}

// grid (H, B T), block HD: out = shr(p.V, 20) and the head's bit length. 8.2 us for 256 rows of 40 heads of 128 (21 MB)
template <int HD>
__global__ __launch_bounds__(HD) void k_tree_out(TreeArgs A, TreeWork W, int64_t* __restrict__ out, int32_t* __restrict__ obits) {
  __shared__ int red[16];
  const int h = blockIdx.x, r = blockIdx.y, d = threadIdx.x, bt = r / A.T, kh = h / A.G;
  const int64_t row = ((int64_t)bt * A.KV + kh) * A.MP + (r - bt * A.T) * A.G + h - kh * A.G;
  const int64_t o = shr64((int64_t)W.acc[row * HD + d], 20);
  out[((int64_t)r * A.H + h) * HD + d] = o;
  if (!obits) return;
  const int m = block_max_i32(bitlen64(abs64(o)), red);
  if (d == 0) obits[(int64_t)r * A.H + h] = m;
}

static bool tree_takes(int B, int T, int H, int KV, int hd, int keys) {
  return B > 0 && T > 0 && T <= TREE_T && H > 0 && KV > 0 && H % KV == 0 && (hd == 64 || hd == 128) && keys > 0 && keys <= TREE_SMAX &&
         (int64_t)B * T <= 65535 && H + 2LL * KV <= 65535 && (int64_t)B * KV <= 65535 && (int64_t)T * (H / KV) <= 65535;
}

static void tree_sizes(TreeArgs& A, int B, int T, int H, int KV, int keys) {
  A.B = B, A.T = T, A.H = H, A.KV = KV, A.G = H / KV, A.keys = keys;
  A.M = T * A.G;
  A.MP = (int)cdiv(A.M, 16) * 16;
  A.NG = (int)cdiv(keys, TREE_KG);
  A.Sp = cdiv(keys, TREE_CK) * TREE_CK;
}

// the parts of the workspace, each a multiple of 16 bytes long; its bytes
static int64_t tree_work(const TreeArgs& A, int hd, int8_t* at, TreeWork& W) {
  const int64_t rows = (int64_t)A.B * A.KV * A.MP, off0 = 0;
  int64_t off = off0;
  auto take = [&](int64_t bytes) {
    int8_t* p = at ? at + off : nullptr;
    off += (bytes + 15) / 16 * 16;
    return p;
  };
  W.d = reinterpret_cast<uint32_t*>(take(rows * A.Sp * 4));
  W.acc = reinterpret_cast<uint64_t*>(take(rows * hd * 8));
  W.cm = reinterpret_cast<int64_t*>(take(rows * A.NG * 8));
  W.es = reinterpret_cast<int64_t*>(take(rows * 8));
  W.qd = take(rows * 2 * hd);
  W.shq = reinterpret_cast<int32_t*>(take(rows * 4));
  W.qsum = reinterpret_cast<int32_t*>(take(rows * 4));
  W.neg = reinterpret_cast<int32_t*>(take(rows * 4));
  W.seq = reinterpret_cast<TreeSeq*>(take(A.B * sizeof(TreeSeq)));
  return off;
}

// How k_tree_pv is split: row groups of mt tiles, runs of keys. A block, one a CU, takes about 5 us and 2 + 0.8 mt a step of 128 keys, and
// the totals' atomics 8 ns each; the cheapest of all numbers of tiles and of up to four rounds of blocks (256 CUs) is taken. us a layer, 28
// heads over 4 of 128 at 1793 positions, a tree of 26: 1 tile in 5 runs (taken) 36.3, 2 in 10 36.0, 3 in 8 37.0, 3 in 15 37.8; 40 over 8 at
// 6001, four trees of 64: 5 tiles in 2 runs (taken) 321, 3 in 5 394, 2 in 5 463, 1 in 5 569.
// Heads of 64 have no term of their own: 14 over 2, four trees of 64 at 6001: 5 tiles in 5 runs (taken) 107, 3 in 3 108, 2 in 2 115, 1 in
// 1 140; a tree of 26 at 1793: 2 in 15 (taken) 28.3, 2 in 8 26.3, 1 in 8 25.6.
struct TreeSplit {
  int mt, groups, ksplit;
};
static TreeSplit tree_split(const TreeArgs& A, int hd) {
  const int64_t seqs = (int64_t)A.B * A.KV, tiles = cdiv(A.M, 16), steps = A.Sp / TREE_CK, least = cdiv(A.keys, 32768);
  TreeSplit best = {1, (int)tiles, (int)std::max(least, std::min<int64_t>(steps, 1))};
  double cost = 1e30;
  for (int most = 1; most <= TREE_MT; ++most) {
    const int64_t groups = cdiv(tiles, most);
    const int mt = (int)cdiv(tiles, groups);
    for (int rounds = 1; rounds <= 4; ++rounds) {
      const int64_t ks = std::max(least, std::min(steps, std::max<int64_t>(1, 256 * rounds / (groups * seqs))));
      const double c = (double)cdiv(groups * seqs * ks, 256) * (5 + (double)cdiv(steps, ks) * (2 + 0.8 * mt)) + 8e-6 * ks * A.M * hd * seqs;
      if (c < cost) cost = c, best = {mt, (int)groups, (int)ks};
    }
  }
  return best;
}

template <int HD>
static void tree_go(int64_t* t, const int32_t* s, const int64_t* b, const int64_t* cos_t, const int64_t* sin_t, int16_t* kq,
                    int32_t* sk, int64_t* v, const int32_t* exp_t, int64_t* out, int32_t* obits, const TreeArgs& A,
                    const TreeWork& W, int INV, int clear_t, hipStream_t st) {
  hipLaunchKernelGGL((k_tree_qkv<HD>), dim3(A.B * A.T, A.H + 2 * A.KV), dim3(64), 0, st, t, s, b, cos_t, sin_t, kq, sk, v, A, W, clear_t);
  const int64_t seqs = (int64_t)A.B * A.KV;
  if (A.keys <= TREE_SHORT || (A.keys <= 2 * TREE_SHORT && (int64_t)A.B * A.T * A.H >= TREE_SHORT_ROWS)) {
    const dim3 g((uint32_t)seqs, (uint32_t)cdiv(A.M, 16));
    auto k = A.keys <= TREE_SHORT ? k_tree_short<HD, 1> : k_tree_short<HD, 2>;
    hipLaunchKernelGGL(k, g, dim3(512), 0, st, kq, sk, v, exp_t, A, W, INV, out, obits);
    return;
  }
  const int mparts = (int)std::min(cdiv(A.M, 64), std::max<int64_t>(1, 1024 / (A.NG * seqs)));
  hipLaunchKernelGGL((k_tree_scores<HD>), dim3(A.NG * mparts, A.KV, A.B), dim3(256), 0, st, kq, sk, A, W, INV, mparts);
  hipLaunchKernelGGL((k_tree_exp<HD>), dim3(A.M, A.KV, A.B), dim3(256), 0, st, exp_t, A, W);
  const TreeSplit sp = tree_split(A, HD);
  const int mt = sp.mt;
  const dim3 pv((uint32_t)seqs, sp.groups, sp.ksplit);
  switch (mt) {
    case 1: hipLaunchKernelGGL((k_tree_pv<HD, 1>), pv, dim3(512), 0, st, v, A, W); break;
    case 2: hipLaunchKernelGGL((k_tree_pv<HD, 2>), pv, dim3(512), 0, st, v, A, W); break;
    case 3: hipLaunchKernelGGL((k_tree_pv<HD, 3>), pv, dim3(512), 0, st, v, A, W); break;
    case 4: hipLaunchKernelGGL((k_tree_pv<HD, 4>), pv, dim3(512), 0, st, v, A, W); break;
    default: hipLaunchKernelGGL((k_tree_pv<HD, 5>), pv, dim3(512), 0, st, v, A, W); break;
  }
  hipLaunchKernelGGL((k_tree_out<HD>), dim3(A.H, A.B * A.T), dim3(HD), 0, st, A, W, out, obits);
}

}  // namespace exact

using namespace exact;

extern "C" int64_t exact_attention_tree_workspace(int32_t B, int32_t T, int32_t H, int32_t KV, int32_t hd, int32_t keys) {
  if (!tree_takes(B, T, H, KV, hd, keys)) return 0;
  TreeArgs A;
  TreeWork W;
  tree_sizes(A, B, T, H, KV, keys);
  return tree_work(A, hd, nullptr, W);
}

extern "C" int exact_attention_tree(int64_t* t, const int32_t* s, const int64_t* b, const int64_t* cos_t, const int64_t* sin_t,
                                    int32_t rope_n, const int32_t* slot, const int32_t* base, const int32_t* depth,
                                    const int64_t* mask, const int32_t* nodes, int16_t* kq, int32_t* sk, int64_t* v,
                                    int32_t nslots, const int32_t* exp_t, int64_t* out, int32_t* obits, void* work,
                                    int64_t work_bytes, int32_t B, int32_t T, int32_t H, int32_t KV, int32_t hd, int32_t Smax,
                                    int32_t keys, int32_t INV, int32_t clear_t, void* stream) {
  if (!t || !s || !cos_t || !sin_t || !slot || !base || !depth || !mask || !kq || !sk || !v || !exp_t || !out || !work)
    return EXACT_E_ARG;
  if (B <= 0 || T <= 0 || H <= 0 || KV <= 0 || H % KV || hd <= 0 || Smax <= 0 || keys <= 0 || keys > Smax || rope_n <= 0 || nslots <= 0)
    return EXACT_E_ARG;
  if (!tree_takes(B, T, H, KV, hd, keys)) return EXACT_E_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(work) & 255) || work_bytes < exact_attention_tree_workspace(B, T, H, KV, hd, keys))
    return EXACT_E_ARG;
  if ((reinterpret_cast<uintptr_t>(kq) | reinterpret_cast<uintptr_t>(v) | reinterpret_cast<uintptr_t>(out)) & 15)
    return EXACT_E_UNSUPPORTED;
  TreeArgs A;
  TreeWork W;
  A.slot = slot, A.base = base, A.depth = depth, A.nodes = nodes, A.mask = mask;
  A.nslots = nslots, A.Smax = Smax, A.rope_n = rope_n;
  tree_sizes(A, B, T, H, KV, keys);
  tree_work(A, hd, static_cast<int8_t*>(work), W);
  auto go = hd == 64 ? tree_go<64> : tree_go<128>;
  go(t, s, b, cos_t, sin_t, kq, sk, v, exp_t, out, obits, A, W, INV, clear_t, as_stream(stream));
  return launch_status("attention_tree");
}
