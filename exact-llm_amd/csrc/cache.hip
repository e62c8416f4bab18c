// Rows of the layers' caches moved and copied on the device: one launch for every layer, whose caches lie in one allocation each
// (kq, sk, v: [L][slots][KV][Smax][...]).
#include "exact_common.h"
#include "abi_util.h"

namespace exact {

#define CACHE_NT 256
// rows in flight in k_cache_keep. us for 8 paths of 6, 16 and 56 nodes in 48 layers of 8 heads of 128 with 4 / 8 / 16: 12.8 / 12.6 / 19.4,
// 29.1 / 28.6 / 40.2, 139 / 137 / 187 (registers)
#define CACHE_ROWS 8
#define CACHE_CK 64    // positions a block of k_cache_fork

// grid (units of a position, B, L): a thread owns 16 bytes (or the shift) of one (layer, sequence, KV head)'s rows and moves them from base
// + path[d] to base + d for d = 0, 1, ... An accepted path goes up, so path[d] >= d: a row is read before any row that is written over it,
// and the first CACHE_ROWS rows can be loaded together. A path that does not go up ends there. A sequence whose slot one before it has
// would race: it is left out. Latency of the loads of slots, counts and path, one after the other behind a barrier, and of the rounds of
// CACHE_ROWS rows, up to near the copy rate where many rows move. us in a graph: one path of 1 / 8 / 56 rows in 24 layers of 2 heads of 64
// 4.6 / 7.5 / 38, 8 paths of 1 / 6 / 16 / 56 in 48 layers of 8 heads of 128 5.8 / 12.6 / 28.6 (4.1 TB/s) / 137 (3.2 TB/s).
__global__ __launch_bounds__(CACHE_NT) void k_cache_keep(v4i* __restrict__ kq, int32_t* __restrict__ sk, v4i* __restrict__ v,
                                                         int nslots, const int32_t* __restrict__ slot,
                                                         const int32_t* __restrict__ base, const int32_t* __restrict__ path,
                                                         const int32_t* __restrict__ n, int T, int KV, int hd, int Smax) {
  const int ku = hd / 8, U = ku + hd / 2 + 1;   // 16-byte units of a key, units of a row (the last: its shift)
  const int i = blockIdx.x * CACHE_NT + threadIdx.x, kh = i / U, u = i - kh * U, b = blockIdx.y;
  const int64_t l = blockIdx.z, sl = slot[b], p0 = base[b];
  int again = 0;
  for (int j = threadIdx.x; j < b; j += CACHE_NT) again |= slot[j] == sl && n[j] > 0;
  if (b && __syncthreads_or(again)) return;
  if (kh >= KV || sl < 0 || sl >= nslots || p0 < 0 || p0 >= Smax) return;
  const int nb = min(n[b], T);
  const int64_t row0 = ((l * nslots + sl) * KV + kh) * Smax + p0;
  const int32_t* pb = path + (int64_t)b * T;
  int last = -1;
  for (int d0 = 0; d0 < nb; d0 += CACHE_ROWS) {
    v4i val[CACHE_ROWS];
    int from[CACHE_ROWS];
#pragma unroll
    for (int j = 0; j < CACHE_ROWS; ++j) {
      const int f = d0 + j < nb ? pb[d0 + j] : -1;
      const bool ok = f > last && f < T && p0 + f < Smax;   // after a refused entry no later one is above last
      last = ok ? f : INT32_MAX;
      from[j] = ok && f != d0 + j ? f : -1;
      if (from[j] < 0) continue;
      const int64_t r = row0 + f;
      if (u < ku) val[j] = kq[r * ku + u];
      else if (u < U - 1) val[j] = v[r * (hd / 2) + u - ku];
      else val[j][0] = sk[r];
    }
#pragma unroll
    for (int j = 0; j < CACHE_ROWS; ++j) {
      if (from[j] < 0) continue;
      const int64_t r = row0 + d0 + j;
      if (u < ku) kq[r * ku + u] = val[j];
      else if (u < U - 1) v[r * (hd / 2) + u - ku] = val[j];
      else sk[r] = val[j][0];
    }
  }
}

// grid (chunks of CACHE_CK positions, L KV, pairs): the chunk's rows of one (layer, KV head) from slot src to slot dst, which are
// contiguous in each array. A pair whose dst is a source, or the dst of a pair before it, is left out: it would race. Copy rate: 301 us,
// 5.1 TB/s, for 1793 positions of 28 layers of 4 heads of 128 to three slots; 7.2 us for 137 positions of 24 layers of 2 heads of 64, whose
// 144 blocks leave 112 CUs idle.
__global__ __launch_bounds__(CACHE_NT) void k_cache_fork(v4i* __restrict__ kq, int32_t* __restrict__ sk, v4i* __restrict__ v,
                                                         int nslots, const int32_t* __restrict__ src,
                                                         const int32_t* __restrict__ dst, const int32_t* __restrict__ n, int M,
                                                         int KV, int hd, int Smax, int keys) {
  const int m = blockIdx.z, kh = blockIdx.y % KV, tid = threadIdx.x;
  const int64_t l = blockIdx.y / KV, a = src[m], b = dst[m];
  const int p0 = blockIdx.x * CACHE_CK, p1 = min(min(n[m], keys), p0 + CACHE_CK);
  if (p0 >= p1 || a < 0 || a >= nslots || b < 0 || b >= nslots) return;
  int clash = 0;
  for (int j = tid; j < M; j += CACHE_NT) clash |= src[j] == b || (j < m && dst[j] == b);
  if (__syncthreads_or(clash)) return;
  const int64_t ra = ((l * nslots + a) * KV + kh) * Smax + p0, rb = ((l * nslots + b) * KV + kh) * Smax + p0;
  const int rows = p1 - p0;
  for (int j = tid; j < rows * (hd / 2); j += CACHE_NT) v[rb * (hd / 2) + j] = v[ra * (hd / 2) + j];
  for (int j = tid; j < rows * (hd / 8); j += CACHE_NT) kq[rb * (hd / 8) + j] = kq[ra * (hd / 8) + j];
  for (int j = tid; j < rows; j += CACHE_NT) sk[rb + j] = sk[ra + j];
}

static int cache_check(const void* kq, const void* sk, const void* v, int L, int nslots, int KV, int hd, int Smax) {
  if (!kq || !sk || !v || L <= 0 || nslots <= 0 || KV <= 0 || hd <= 0 || Smax <= 0) return EXACT_E_ARG;
  if (hd % 8 || hd > 1024 || ((uintptr_t)kq | (uintptr_t)v) & 15) return EXACT_E_UNSUPPORTED;
  return EXACT_OK;
}

}  // namespace exact

using namespace exact;

extern "C" int exact_cache_keep(int16_t* kq, int32_t* sk, int64_t* v, int32_t L, int32_t nslots, const int32_t* slot,
                                const int32_t* base, const int32_t* path, const int32_t* n, int32_t B, int32_t T, int32_t KV,
                                int32_t hd, int32_t Smax, void* stream) {
  if (!slot || !base || !path || !n || B <= 0 || T <= 0) return EXACT_E_ARG;
  if (const int rc = cache_check(kq, sk, v, L, nslots, KV, hd, Smax)) return rc;
  if (KV > 65535 || B > 65535 || L > 65535) return EXACT_E_UNSUPPORTED;
  hipLaunchKernelGGL(k_cache_keep, dim3((uint32_t)cdiv(KV * (hd / 8 + hd / 2 + 1), CACHE_NT), B, L), dim3(CACHE_NT), 0,
                     as_stream(stream), reinterpret_cast<v4i*>(kq), sk, reinterpret_cast<v4i*>(v), nslots, slot, base, path, n, T,
                     KV, hd, Smax);
  return launch_status("cache_keep");
}

extern "C" int exact_cache_fork(int16_t* kq, int32_t* sk, int64_t* v, int32_t L, int32_t nslots, const int32_t* src,
                                const int32_t* dst, const int32_t* n, int32_t M, int32_t KV, int32_t hd, int32_t Smax,
                                int32_t keys, void* stream) {
  if (!src || !dst || !n || M <= 0 || keys <= 0 || keys > Smax) return EXACT_E_ARG;
  if (const int rc = cache_check(kq, sk, v, L, nslots, KV, hd, Smax)) return rc;
  if (M > 65535 || (int64_t)L * KV > 65535) return EXACT_E_UNSUPPORTED;
  hipLaunchKernelGGL(k_cache_fork, dim3((uint32_t)cdiv(keys, CACHE_CK), L * KV, M), dim3(CACHE_NT), 0, as_stream(stream),
                     reinterpret_cast<v4i*>(kq), sk, reinterpret_cast<v4i*>(v), nslots, src, dst, n, M, KV, hd, Smax,
                     keys);
  return launch_status("cache_fork");
}
