// Drafted tokens judged by the target model's logits (exact_verify_draft), in the integers of the sampler (exact_llm.py:250-259):
//   p = isoftmax_row(shr(lg * tnum, 16)) (Q20), P = sum p; q (Q20) the draft model's probabilities, Q = sum q
// A token x drafted from q is accepted with probability min(1, (p / P) / (q / Q)): u q(x) P < p(x) Q 2^20 for a u of [0, 2^20).
// After a rejection the token comes from w = max(p Q - q P, 0), which together make the tokens distributed as p / P. Every
// product is below 2^60 (p, q, P, Q <= 2^20), so both are exact in int64; with an exp table with negative entries below 2^63, since a row
// whose p sum to 2^23 or more counts as one without probability.
#include "exact_common.h"
#include "abi_util.h"
#include "sample_ops.h"

namespace exact {

#define VERIFY_K 64   // drafted tokens a sequence
#define VERIFY_V (1 << 30)   // logits a row: chunks end below 2^31

// ---- split over chunks, five launches for rows of many logits: block (c, row) is chunk c of a target row (or of a sequence), a wave
// owns PT * 64 consecutive logits. One block walks a row of 151936 logits four times in 190 us; a launch here starts from the
// chunk results of the one before. The logits are read once: the first launch keeps them as 32-bit distances to their chunk's maximum,
// the second as exponentials, which every later launch reads (74.4 us for 8 sequences of 7 drafts at 152064; made again by each, 78.6).
// The first launch of that call reads 129 MB of logits and q at 4.85 TB/s (6.15 with the distances that it writes), the others 4 bytes a
// logit that the caches hold in part.
#define VERIFY_NT 256
// logits of a row that one block holds: with 8000, one row takes 19.4 us (over chunks 17.0), 9 rows 20.8 (22.3), 160 rows 22.0 (25.1)
#define VERIFY_SHORT 8192

struct VerifyArgs {
  const int64_t *lg, *q;
  const int32_t *tok, *u, *drafted, *T;
  int64_t tnum;
  int32_t *ids, *n;
  int K, V, nch;
  __device__ __forceinline__ int count(int b) const { return drafted ? min(max(drafted[b], 0), K) : K; }
};

struct VerifyWork {
  int64_t *mx, *es, *ps, *qs;   // [B (K + 1)][nch]: of each chunk the maximum, sums of exponentials, of p and of q
  int64_t* ws;                  // [B][nch]: sum of the rest's weights in the row that rejected
  int64_t* at;                  // [B][4]: that row (or the one after the last token), its sum of exponentials, P, Q
  uint32_t* d;                  // [B (K + 1)][V]: maximum of the chunk - logit, then exponentials
};

__device__ __forceinline__ int64_t wave_total(const int64_t* v, int n, int lane) {
  uint64_t s = 0;
  for (int i = lane; i < n; i += 64) s += (uint64_t)v[i];
  return wave_sum64((int64_t)s);
}
__device__ __forceinline__ int64_t wave_top(const int64_t* v, int n, int lane) {
  int64_t m = INT64_MIN;
  for (int i = lane; i < n; i += 64) m = max64(m, v[i]);
  return wave_max64(m);
}

// a row's totals from its chunks', by one wave; the loads of a step are in flight together
struct RowSums {
  int64_t mx, es, P, Q;
};
__device__ __forceinline__ RowSums row_sums(const VerifyWork& W, int64_t r, int nch, int lane) {
  int64_t mx = INT64_MIN, es = 0, P = 0, Q = 0;
  for (int i = lane; i < nch; i += 64) {
    const int64_t a = W.mx[r * nch + i], b = W.es[r * nch + i], c = W.ps[r * nch + i], d = W.qs[r * nch + i];
    mx = max64(mx, a);
    es += b;
    P += c;
    Q += d;
  }
  return {wave_max64(mx), wave_sum64(es), wave_sum64(P), wave_sum64(Q)};
}

// grid (nch, B (K + 1))
template <int PT>
__global__ __launch_bounds__(VERIFY_NT) void k_verify_max(VerifyArgs A, VerifyWork W) {
  __shared__ int64_t red[2][16];
  const int64_t r = blockIdx.y;
  const int b = (int)(r / (A.K + 1)), i = (int)(r - (int64_t)b * (A.K + 1)), d = A.count(b);
  if (i > d) return;
  const int j0 = blockIdx.x * (PT * VERIFY_NT) + (threadIdx.x >> 6) * (PT * 64) + (threadIdx.x & 63);
  const int64_t* row = A.lg + r * A.V;
  int64_t a[PT], m = INT64_MIN, Q = 0;
#pragma unroll
  for (int k = 0; k < PT; ++k) a[k] = j0 + 64 * k < A.V ? row[j0 + 64 * k] : 0;
  if (i < d) {
    const int64_t* qr = A.q + ((int64_t)b * A.K + i) * A.V;
#pragma unroll
    for (int k = 0; k < PT; ++k) Q += j0 + 64 * k < A.V ? qr[j0 + 64 * k] : 0;
  }
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    a[k] = j0 + 64 * k < A.V ? shr64(a[k] * A.tnum, EXACT_F) : INT64_MIN;
    m = max64(m, a[k]);
  }
  m = block_max64_1(m, red[0]);
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    const uint64_t gap = (uint64_t)m - (uint64_t)a[k];
    if (j0 + 64 * k < A.V) W.d[r * A.V + j0 + 64 * k] = gap < EXP_FAR ? (uint32_t)gap : EXP_FAR;
  }
  if (i < d) Q = block_sum64_1(Q, red[1]);
  if (threadIdx.x == 0) {
    W.mx[r * A.nch + blockIdx.x] = m;
    W.qs[r * A.nch + blockIdx.x] = Q;
  }
}

// grid (nch, B (K + 1)): the exponentials over the distances, and their sum
template <int PT>
__global__ __launch_bounds__(VERIFY_NT) void k_verify_exp(VerifyArgs A, VerifyWork W) {
  __shared__ int64_t red[16];
  const int64_t r = blockIdx.y;
  const int b = (int)(r / (A.K + 1));
  if (r - (int64_t)b * (A.K + 1) > A.count(b)) return;
  const int j0 = blockIdx.x * (PT * VERIFY_NT) + (threadIdx.x >> 6) * (PT * 64) + (threadIdx.x & 63);
  uint32_t* d = W.d + r * A.V;
  uint32_t x[PT];
#pragma unroll
  for (int k = 0; k < PT; ++k) x[k] = j0 + 64 * k < A.V ? d[j0 + 64 * k] : EXP_FAR;
  const int64_t cm = W.mx[r * A.nch + blockIdx.x];
  const uint32_t gap = exp_gap(wave_top(W.mx + r * A.nch, A.nch, threadIdx.x & 63), cm);
  int64_t es = 0;
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    const int32_t e = lut_exp_kept(A.T, gap, x[k]);
    es += e;
    if (j0 + 64 * k < A.V) d[j0 + 64 * k] = (uint32_t)e;
  }
  es = block_sum64_1(es, red);
  if (threadIdx.x == 0) W.es[r * A.nch + blockIdx.x] = es;
}

// the lane's exponentials of row r
template <int PT>
__device__ __forceinline__ void verify_kept(const VerifyArgs& A, const VerifyWork& W, int64_t r, int32_t (&e)[PT]) {
  const int j0 = blockIdx.x * (PT * VERIFY_NT) + (threadIdx.x >> 6) * (PT * 64) + (threadIdx.x & 63);
#pragma unroll
  for (int k = 0; k < PT; ++k) e[k] = j0 + 64 * k < A.V ? (int32_t)W.d[r * A.V + j0 + 64 * k] : 0;
}

// grid (nch, B (K + 1))
template <int PT>
__global__ __launch_bounds__(VERIFY_NT) void k_verify_psum(VerifyArgs A, VerifyWork W) {
  __shared__ int64_t red[16];
  const int64_t r = blockIdx.y;
  const int b = (int)(r / (A.K + 1)), lane = threadIdx.x & 63;
  if (r - (int64_t)b * (A.K + 1) > A.count(b)) return;
  int32_t e[PT];
  verify_kept(A, W, r, e);
  const RowSums R = row_sums(W, r, A.nch, lane);
  const int64_t es = R.es;
  const double es20 = sum20(es), rb = sum20_rcp(es20);
  int64_t P = 0;
#pragma unroll
  for (int k = 0; k < PT; ++k) P += prob20(e[k], es, es20, rb);
  P = block_sum64_1(P, red);
  if (threadIdx.x == 0) W.ps[r * A.nch + blockIdx.x] = P;
}

// grid (nch, B): every block judges the sequence's tokens (a wave a row), then sums the rest's weights of its chunk of the row that
// rejected; the first block writes the accepted tokens
template <int PT>
__global__ __launch_bounds__(VERIFY_NT) void k_verify_rest(VerifyArgs A, VerifyWork W) {
  __shared__ int64_t red[16];
  __shared__ RowSums rows[VERIFY_K + 1];
  __shared__ int ok[VERIFY_K + 1];
  const int b = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = A.count(b), nch = A.nch;
  const int64_t r0 = (int64_t)b * (A.K + 1);
  for (int i = wave; i <= d; i += VERIFY_NT / 64) {
    const int64_t r = r0 + i;
    const int x = i < d ? A.tok[(int64_t)b * A.K + i] : -1;
    const bool in = x >= 0 && x < A.V;
    const int64_t qx = in ? A.q[((int64_t)b * A.K + i) * A.V + x] : 0;
    const int32_t ex = in ? (int32_t)W.d[r * A.V + x] : 0;
    const int u = A.u[r];
    RowSums R = row_sums(W, r, nch, lane);
    if (R.P >= PROB_NONE) R.es = R.P = 0;
    const double es20 = sum20(R.es);
    if (lane == 0) {
      rows[i] = R;
      ok[i] = in && verify_accepts(u, prob20(ex, R.es, es20, sum20_rcp(es20)), R.P, qx, R.Q);
    }
  }
  __syncthreads();
  int a = 0;
  while (a < d && ok[a]) ++a;
  const RowSums R = rows[a];
  if (a < d) {
    const int j0 = blockIdx.x * (PT * VERIFY_NT) + wave * (PT * 64) + lane;
    const int64_t* qr = A.q + ((int64_t)b * A.K + a) * A.V;
    const double es20 = sum20(R.es), rb = sum20_rcp(es20);
    int32_t e[PT];
    verify_kept(A, W, r0 + a, e);
    int64_t qv[PT], ws = 0;
#pragma unroll
    for (int k = 0; k < PT; ++k) qv[k] = j0 + 64 * k < A.V ? qr[j0 + 64 * k] : 0;
#pragma unroll
    for (int k = 0; k < PT; ++k)
      if (j0 + 64 * k < A.V) ws += verify_rest(prob20(e[k], R.es, es20, rb), R.P, qv[k], R.Q);
    ws = block_sum64_1(ws, red);
    if (threadIdx.x == 0) W.ws[(int64_t)b * nch + blockIdx.x] = ws;
  }
  if (blockIdx.x) return;
  for (int i = threadIdx.x; i <= A.K; i += VERIFY_NT) A.ids[r0 + i] = i < a ? A.tok[(int64_t)b * A.K + i] : (i == a ? A.V : -1);
  if (threadIdx.x == 0) {
    A.n[b] = a;
    int64_t* at = W.at + 4LL * b;
    at[0] = a, at[1] = R.es, at[2] = R.P, at[3] = R.Q;
  }
}

// A block's prefix sums above the target, of the lanes' weights w (their sum s; weight k is real for 64 k < left) on top of carry.
template <int PT, int NT>
__device__ __forceinline__ int verify_above(const int64_t (&w)[PT], int64_t s, int64_t carry, int64_t target, int left) {
  __shared__ int64_t wsum[NT / 64];
  __shared__ int over[NT / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  s = wave_sum64(s);
  if (lane == 0) wsum[wave] = s;
  __syncthreads();
  for (int i = 0; i < wave; ++i) carry += wsum[i];
  int above = 0;
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    const int64_t p = carry + wave_incl_scan64(w[k], lane);
    above += __popcll(__ballot(64 * k < left && p > target));
    carry = readlane64(p, 63);
  }
  if (lane == 0) over[wave] = above;
  __syncthreads();
  above = 0;
  for (int i = 0; i < NT / 64; ++i) above += over[i];
  return above;
}

// grid (nch, B): the one chunk in which the weights' sums pass the target counts those up to it (no chunk if all weights are 0)
template <int PT>
__global__ __launch_bounds__(VERIFY_NT) void k_verify_pick(VerifyArgs A, VerifyWork W) {
  const int b = blockIdx.y, c = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nch = A.nch;
  const int64_t *at = W.at + 4LL * b, r0 = (int64_t)b * (A.K + 1);
  const int a = (int)at[0];
  const int64_t r = r0 + a, es = at[1], P = at[2], Q = at[3];
  const int64_t* sums = W.ws + (int64_t)b * nch;
  int64_t total = a < A.count(b) ? wave_total(sums, nch, lane) : 0;
  const bool rest = total > 0;
  if (!rest) sums = W.ps + r * nch, total = P;
  if (total == 0) return;
  int64_t carry = wave_total(sums, c, lane);
  const int64_t target = verify_target(A.u[r0 + A.K], total);
  if (target < carry || target >= carry + sums[c]) return;
  const int j0 = c * (PT * VERIFY_NT) + wave * (PT * 64) + lane;
  const int64_t* qr = A.q + ((int64_t)b * A.K + a) * A.V;   // read for a < d only
  const double es20 = sum20(es), rb = sum20_rcp(es20);
  int32_t e[PT];
  verify_kept(A, W, r, e);
  int64_t w[PT], s = 0;
#pragma unroll
  for (int k = 0; k < PT; ++k) {
    w[k] = prob20(e[k], es, es20, rb);
    if (rest) w[k] = j0 + 64 * k < A.V ? verify_rest(w[k], P, qr[j0 + 64 * k], Q) : 0;
    s += w[k];
  }
  const int above = verify_above<PT, VERIFY_NT>(w, s, carry, target, A.V - j0);
  if (threadIdx.x == 0) A.ids[r] = (int32_t)(min((c + 1) * (PT * VERIFY_NT), A.V) - above);
}

// ---- rows of up to VERIFY_SHORT logits, two launches: a block holds a row in registers, 512 consecutive logits a wave. Their time is
// the latency of a chain of loads and barriers, so every load that a launch can start at once starts at once: 6.4 and 5.3 us for 2 rows
// of 1000 logits, no more for 64 of 2000. One block a sequence that walks its rows: 13.5 us, and 61 for 8 sequences of 7 drafts at 2000.
struct VerifyShort {
  int64_t* at;   // [B (K + 1)][4]: a row's sums of exponentials, of p and of q, and whether its token is accepted
  int32_t* e;    // [B (K + 1)][V]: its exponentials
};

// grid B (K + 1): row r's exponentials and sums
template <int NT>
__global__ __launch_bounds__(NT) void k_verify_row(VerifyArgs A, VerifyShort W) {
  __shared__ int64_t red[4][16], px;
  const int64_t r = blockIdx.x;
  const int b = (int)(r / (A.K + 1)), i = (int)(r - (int64_t)b * (A.K + 1)), d = A.count(b);
  const int j0 = (threadIdx.x >> 6) * 512 + (threadIdx.x & 63);
  const bool has = i < A.K;   // a drafted token, its q
  const int64_t* qr = A.q + ((int64_t)b * A.K + i) * A.V;
  int64_t a[8], m = INT64_MIN, Q = 0, P = 0, es = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    a[k] = j0 + 64 * k < A.V ? A.lg[r * A.V + j0 + 64 * k] : 0;
    Q += has && j0 + 64 * k < A.V ? qr[j0 + 64 * k] : 0;
  }
  const int x = has ? A.tok[(int64_t)b * A.K + i] : -1, u = A.u[r];
  const bool in = x >= 0 && x < A.V;
  const int64_t qx = in ? qr[x] : 0;
  if (i > d) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    a[k] = j0 + 64 * k < A.V ? shr64(a[k] * A.tnum, EXACT_F) : INT64_MIN;
    m = max64(m, a[k]);
  }
  m = block_max64_1(m, red[0]);
  int32_t e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    e[k] = j0 + 64 * k < A.V ? (int32_t)lut_exp(A.T, m, a[k]) : 0;
    if (j0 + 64 * k < A.V) W.e[r * A.V + j0 + 64 * k] = e[k];
    es += e[k];
  }
  es = block_sum64_1(es, red[1]);
  const double es20 = sum20(es), rb = sum20_rcp(es20);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int64_t p = prob20(e[k], es, es20, rb);
    P += p;
    if (j0 + 64 * k == x) px = p;
  }
  P = wave_sum64(P);
  Q = wave_sum64(Q);
  if ((threadIdx.x & 63) == 0) red[2][threadIdx.x >> 6] = P, red[3][threadIdx.x >> 6] = Q;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < NT / 64; ++w) P += red[2][w], Q += red[3][w];
  const bool none = P >= PROB_NONE;
  int64_t* at = W.at + 4 * r;
  at[0] = none ? 0 : es;
  at[1] = none ? 0 : P;
  at[2] = Q;
  at[3] = in && !none && verify_accepts(u, px, P, qx, Q);
}

// grid B: the first row whose token is rejected (or the one after the last token), the rest's weights there and the token picked by them
template <int NT>
__global__ __launch_bounds__(NT) void k_verify_end(VerifyArgs A, VerifyShort W) {
  __shared__ int64_t red[16];
  const int b = blockIdx.x, lane = threadIdx.x & 63, d = A.count(b), j0 = (threadIdx.x >> 6) * 512 + lane;
  const int64_t r0 = (int64_t)b * (A.K + 1);
  const bool no = lane < A.K && !W.at[4 * (r0 + lane) + 3];
  const int u = A.u[r0 + A.K];
  const uint64_t left = __ballot(no && lane < d);
  const int a = left ? __builtin_ctzll(left) : d;
  const int64_t r = r0 + a, es = W.at[4 * r], P = W.at[4 * r + 1], Q = W.at[4 * r + 2];
  const int64_t* qr = A.q + ((int64_t)b * A.K + a) * A.V;   // read for a < d only
  int64_t w[8], qv[8], rs = 0, ps = 0;
  int32_t e[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    e[k] = j0 + 64 * k < A.V ? W.e[r * A.V + j0 + 64 * k] : 0;
    qv[k] = a < d && j0 + 64 * k < A.V ? qr[j0 + 64 * k] : 0;
  }
  const double es20 = sum20(es), rb = sum20_rcp(es20);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    w[k] = prob20(e[k], es, es20, rb);
    ps += w[k];
    qv[k] = a < d && j0 + 64 * k < A.V ? verify_rest(w[k], P, qv[k], Q) : 0;
    rs += qv[k];
  }
  const int64_t total = block_sum64_1(rs, red);
  if (total > 0) {
#pragma unroll
    for (int k = 0; k < 8; ++k) w[k] = qv[k];
    ps = rs;
  }
  const int64_t target = verify_target(u, total > 0 ? total : P);
  const int id = A.V - verify_above<8, NT>(w, ps, 0, target, A.V - j0);
  for (int i = threadIdx.x; i <= A.K; i += NT) A.ids[r0 + i] = i < a ? A.tok[(int64_t)b * A.K + i] : (i == a ? id : -1);
  if (threadIdx.x == 0) A.n[b] = a;
}

// the parts of the workspace; its bytes
static int64_t verify_work(int64_t B, int64_t K, int64_t V, int64_t nch, int64_t* at, VerifyWork& W) {
  const int64_t R = B * (K + 1), n = R * nch;
  W = {at, at + n, at + 2 * n, at + 3 * n, at + 4 * n, at + 4 * n + B * nch, (uint32_t*)(at + 4 * n + B * nch + 4 * B)};
  return (4 * n + B * nch + 4 * B) * 8 + R * V * 4;
}
// Logits a lane of the launches over chunks: 4 make more, shorter blocks, 8 half the chunk results. us with 4 and 8: one sequence of 4
// drafts at 151936 27.5 and 29.8, 160 rows of 32000 48.6 and 50.4, 64 rows of 128256 71.1 and 67.5, of 151936 85.9 and 79.2.
static int verify_pt(int64_t B, int64_t K, int64_t V) { return B * (K + 1) * V < 6000000 ? 4 : 8; }

template <int NT>
static void verify_short(const VerifyArgs& A, int64_t* at, int32_t B, hipStream_t st) {
  const VerifyShort W = {at, (int32_t*)(at + 4LL * B * (A.K + 1))};
  hipLaunchKernelGGL((k_verify_row<NT>), dim3(B * (A.K + 1)), dim3(NT), 0, st, A, W);
  hipLaunchKernelGGL((k_verify_end<NT>), dim3(B), dim3(NT), 0, st, A, W);
}
template <int PT>
static void verify_long(const VerifyArgs& A, const VerifyWork& W, int32_t B, hipStream_t st) {
  const dim3 rows(A.nch, B * (A.K + 1)), seqs(A.nch, B), nt(VERIFY_NT);
  hipLaunchKernelGGL((k_verify_max<PT>), rows, nt, 0, st, A, W);
  hipLaunchKernelGGL((k_verify_exp<PT>), rows, nt, 0, st, A, W);
  hipLaunchKernelGGL((k_verify_psum<PT>), rows, nt, 0, st, A, W);
  hipLaunchKernelGGL((k_verify_rest<PT>), seqs, nt, 0, st, A, W);
  hipLaunchKernelGGL((k_verify_pick<PT>), seqs, nt, 0, st, A, W);
}

// One wave a sequence, a lane a node: from the root on, the first child whose token is the target's. Nothing but latency: 1.7 us for a
// tree, 2.8 for 64 trees of 64.
__global__ __launch_bounds__(64) void k_tree_accept(const int32_t* __restrict__ nxt, const int32_t* __restrict__ tok,
                                                    const int32_t* __restrict__ parent, const int32_t* __restrict__ nodes,
                                                    int32_t* __restrict__ path, int32_t* __restrict__ ids,
                                                    int32_t* __restrict__ n, int T) {
  const int lane = threadIdx.x;
  const int64_t row = (int64_t)blockIdx.x * T;
  const int nn = nodes ? nodes[blockIdx.x] : T;
  const bool real = lane < T && lane < nn;
  const int nx = real ? nxt[row + lane] : 0, tk = real ? tok[row + lane] : 0, pa = real && lane ? parent[row + lane] : -1;
  int way = -1, id = -1, cnt = 0;   // lane d: the path's node d and the token after it
  if (nn > 0) {
    int cur = 0;
    for (;;) {   // nodes only go up: at most T steps
      const int want = __builtin_amdgcn_readlane(nx, cur);
      if (lane == cnt) way = cur, id = want;
      ++cnt;
      const uint64_t child = __ballot(pa == cur && lane > cur && tk == want);
      if (!child) break;
      cur = __builtin_ctzll(child);
    }
  }
  if (lane < T) {
    path[row + lane] = way;
    if (ids) ids[row + lane] = id;
  }
  if (lane == 0) n[blockIdx.x] = cnt;
}

}  // namespace exact

using namespace exact;

extern "C" int64_t exact_verify_draft_workspace(int32_t B, int32_t K, int32_t V) {
  VerifyWork W;
  if (B <= 0 || K < 0 || K > VERIFY_K || V <= 0 || V > VERIFY_V) return 0;
  if (V <= VERIFY_SHORT) return (int64_t)B * (K + 1) * (32 + 4LL * V);
  return verify_work(B, K, V, cdiv(V, verify_pt(B, K, V) * VERIFY_NT), nullptr, W);
}

extern "C" int exact_verify_draft(const int64_t* lg, const int64_t* q, const int32_t* tok, const int32_t* u, const int32_t* drafted,
                                  int64_t tnum, const int32_t* exp_t, int32_t* ids, int32_t* n, void* work, int64_t work_bytes,
                                  int32_t B, int32_t K, int32_t V, void* stream) {
  if (!lg || !u || !exp_t || !ids || !n || !work || B <= 0 || K < 0 || V <= 0 || tnum <= 0 || (K && (!q || !tok))) return EXACT_E_ARG;
  if (K > VERIFY_K || V > VERIFY_V || (int64_t)B * (K + 1) > 65535) return EXACT_E_UNSUPPORTED;
  if ((uintptr_t)work % 8 || work_bytes < exact_verify_draft_workspace(B, K, V)) return EXACT_E_ARG;
  const hipStream_t st = as_stream(stream);
  int64_t* at = static_cast<int64_t*>(work);
  const int pt = verify_pt(B, K, V);
  const VerifyArgs A = {lg, q, tok, u, drafted, exp_t, tnum, ids, n, K, V, (int)cdiv(V, pt * VERIFY_NT)};
  VerifyWork W;
  if (V <= 2048) verify_short<256>(A, at, B, st);
  else if (V <= VERIFY_SHORT) verify_short<1024>(A, at, B, st);
  else {
    verify_work(B, K, V, A.nch, at, W);
    if (pt == 4) verify_long<4>(A, W, B, st);
    else verify_long<8>(A, W, B, st);
  }
  return launch_status("verify_draft");
}

extern "C" int exact_tree_accept(const int32_t* nxt, const int32_t* tok, const int32_t* parent, const int32_t* nodes, int32_t* path,
                                 int32_t* ids, int32_t* n, int32_t B, int32_t T, void* stream) {
  if (!nxt || !tok || !parent || !path || !n || B <= 0 || T <= 0) return EXACT_E_ARG;
  if (T > 64) return EXACT_E_UNSUPPORTED;
  hipLaunchKernelGGL(k_tree_accept, dim3(B), dim3(64), 0, as_stream(stream), nxt, tok, parent, nodes, path, ids, n, T);
  return launch_status("tree_accept");
}
