// Log probabilities of given tokens, the entropy of each row's distribution
// and its most likely tokens, from a matrix of logits.
//
//   m = max_i x_i,  l = sum_i e^(x_i - m)
//   log p_i = x_i - m - ln l,   H = ln l - (1 / l) sum_i (x_i - m) e^(x_i - m)
//
// Every term of H is >= 0, so nothing cancels; one of the largest logits is
// left out of l (ln l = log1p of the others), so that the entropy of a sure
// row keeps its digits. Bound by reading the logits once.
//
// One pass: a warp streams batches of 32 x 4 x 16 bytes, and each lane keeps
// the maximum and the sums of what it has seen, rescaled where the maximum
// rises -- no lane waits for another. A lane also leaves the maximum of each
// of its batches in shared memory: the `top` largest logits lie in the few
// lane batches whose maximum reaches t, the top-th largest of 32 group maxima
// (`top` different logits reach t), and only those are read again, from L2.
// Their logits that reach t are placed by counting the larger ones. Where too
// many reach t for that, or fewer than `top` groups have logits at all (masked
// rows, equal logits), only what lies above t is placed by counting, and the
// other places go to the first logits that equal t (1,500 bf16 rows of 151,936,
// 20 places: 111 us; masked but for 3 tokens, with -inf 123, with the type's
// lowest value 127). A row is cut over a cluster of up to 16 CTAs where the rows
// alone do not fill the GPU; CTA 0 joins the pieces.
#include <cooperative_groups.h>

#include <cmath>
#include <cstdint>

#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace orx {
namespace {

constexpr int kLpThreads = 256;
constexpr int kLpCand = 512;      // candidates of a piece that are placed by counting
constexpr int kLpMaxCluster = 16;
constexpr int kLpMaxTop = 32;
constexpr int kLpFew = 256;       // lane batches that are ranked against one another

// Numbers that are in the order of the values (but -0 below +0), and back.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t u) {
  return __uint_as_float((u & 0x80000000u) ? (u & 0x7FFFFFFFu) : ~u);
}
// Order of the alternatives: by value (NaN below everything, -0 equal to +0),
// equal values by index, lowest first. 0 is below every key.
__device__ __forceinline__ unsigned long long token_key(float v, uint32_t idx) {
  uint32_t u = order_of(v == 0.0f ? 0.0f : v);
  if (v != v) u = 1u;
  return (static_cast<unsigned long long>(u) << 32) | (0xFFFFFFFFu - idx);
}
__device__ __forceinline__ uint32_t key_index(unsigned long long k) {
  return 0xFFFFFFFFu - static_cast<uint32_t>(k);
}
__device__ __forceinline__ float key_value(unsigned long long k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return u == 1u ? NAN : value_of(u);
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <int DT>
struct Vec {
  static constexpr int kBytes = DT == kDtBf16 ? 2 : 4;
  static constexpr int kVals = 16 / kBytes;
};
// The values of 16 bytes of logits.
template <int DT>
__device__ __forceinline__ void unpack16(const uint4& w, float* x) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (DT == kDtBf16) {
      x[2 * i] = bf_lo(r[i]);
      x[2 * i + 1] = bf_hi(r[i]);
    } else {
      x[i] = __uint_as_float(r[i]);
    }
  }
}

// The largest of n 16-byte vectors of logits; NaN if one is.
template <int DT, int U>
__device__ __forceinline__ float vecs_max(const uint4* v) {
  uint32_t w[4 * U];
#pragma unroll
  for (int u = 0; u < U; ++u) w[4 * u] = v[u].x, w[4 * u + 1] = v[u].y, w[4 * u + 2] = v[u].z, w[4 * u + 3] = v[u].w;
  if (DT == kDtBf16) {
#pragma unroll
    for (int n = 2 * U; n > 0; n >>= 1)
#pragma unroll
      for (int i = 0; i < n; ++i) asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(w[i]) : "r"(w[i + n]));
    return max_nan(bf_lo(w[0]), bf_hi(w[0]));
  }
#pragma unroll
  for (int n = 2 * U; n > 0; n >>= 1)
#pragma unroll
    for (int i = 0; i < n; ++i)
      w[i] = __float_as_uint(max_nan(__uint_as_float(w[i]), __uint_as_float(w[i + n])));
  return __uint_as_float(w[0]);
}

struct LpPiece {  // what one CTA knows of its piece of the row
  float m, l, e;  // maximum; sums over the logits below it, relative to it
  int n;          // logits equal to it
  int pad;
  unsigned long long keys[kLpMaxTop];  // its largest, in order; 0 behind the last
};

constexpr int kLpList = 512;      // lane batches that are read again

struct LpShared {
  LpPiece piece[kLpMaxCluster];  // of CTA 0: written by their CTAs
  alignas(16) float group_max[32];
  float red_l[8], red_e[8];
  float thr;
  int red_n[8], count, listed;
  unsigned long long red_k[8];
  unsigned long long cand[kLpCand];
  int list[kLpList];
  // the maxima of all lane batches follow, [batch][lane]
};

// U: 16-byte vectors of a lane in a batch.
template <int DT, int U>
__global__ void __launch_bounds__(kLpThreads, 4) logprobs_kernel(LogprobArgs a, int piece_batches) {
  constexpr int B = Vec<DT>::kBytes, N = Vec<DT>::kVals, W = kLpThreads / 32;
  constexpr float kLog2e = 1.4426950408889634f;
  extern __shared__ __align__(16) uint8_t lp_raw[];
  LpShared& sm = *reinterpret_cast<LpShared*>(lp_raw);
  float* maxima = reinterpret_cast<float*>(lp_raw + sizeof(LpShared));
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = static_cast<int>(cluster.block_rank());
  const int pieces = static_cast<int>(cluster.num_blocks());
  const long long row = blockIdx.x / pieces;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  // The row as whole 16-byte vectors; what the first and the last have outside the row is -inf.
  const uint8_t* base = static_cast<const uint8_t*>(a.logits) + row * a.row_stride * B;
  const int lead = static_cast<int>(reinterpret_cast<uintptr_t>(base) & 15) / B;
  const uint4* vec = reinterpret_cast<const uint4*>(base - lead * B);
  const int vecs = (lead + a.vocab + N - 1) / N;
  const int whole0 = lead ? 1 : 0, whole1 = (lead + a.vocab) / N;  // vectors [whole0, whole1) lie inside
  const int batches = (vecs + 32 * U - 1) / (32 * U);
  const int b0 = min(batches, rank * piece_batches), b1 = min(batches, b0 + piece_batches);

  auto load1 = [&](int v) {
    if (v >= whole0 && v < whole1) return __ldg(vec + v);
    uint32_t r[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (DT == kDtBf16) {
        uint32_t h[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const int i = v * N + 2 * j + y - lead;
          h[y] = i >= 0 && i < a.vocab ? reinterpret_cast<const uint16_t*>(base)[i] : 0xFF80u;
        }
        r[j] = h[0] | (h[1] << 16);
      } else {
        const int i = v * N + j - lead;
        r[j] = i >= 0 && i < a.vocab ? reinterpret_cast<const uint32_t*>(base)[i] : 0xFF800000u;
      }
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
  };
  auto load = [&](int b, uint4* x) {
    const int v = b * 32 * U + lane;
    if (b * 32 * U >= whole0 && (b + 1) * 32 * U <= whole1) {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = __ldg(vec + v + 32 * u);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = load1(v + 32 * u);
    }
  };

  if (t == 0) sm.count = sm.listed = 0;
  if (rank == 0)
    for (int i = t; i < pieces * kLpMaxTop; i += kLpThreads)
      sm.piece[i / kLpMaxTop].keys[i % kLpMaxTop] = 0;
  if (pieces > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  LpPiece* out = cluster.map_shared_rank(&sm.piece[rank], 0);
  int target = -1;
  float target_x = 0.f;
  if (rank == 0 && t == 0 && a.logprob) {
    target = a.targets[row];
    if (target >= 0 && target < a.vocab)
      target_x = DT == kDtBf16 ? bf2f(reinterpret_cast<const uint16_t*>(base)[target])
                               : reinterpret_cast<const float*>(base)[target];
    else
      target = -1;
  }

  // ---- the pass ----
  float m = -INFINITY, e = 0.f;
  float rest = 0.f, last = 0.f;  // sums of p over the batches but the maximum's, and over that
  int held = -1;
  uint4 next[U];
  if (b0 + warp < b1) load(b0 + warp, next);
  for (int b = b0 + warp; b < b1; b += W) {
    uint4 cur[U];
#pragma unroll
    for (int u = 0; u < U; ++u) cur[u] = next[u];
    if (b + W < b1) load(b + W, next);
    const float bm = vecs_max<DT, U>(cur);
    maxima[(b - b0) * 32 + lane] = bm;
    const bool rise = !(bm <= m);  // with NaN too, which the maximum keeps
    const float nm = max_nan(m, bm), mm = nm == -INFINITY ? 0.f : nm;
    // no further than where f is 0 anyhow, so that a rise from the type's lowest value is no 0 * inf
    const float down = max_nan(m - mm, -1e5f), f = rise ? ex2(down * kLog2e) : 1.0f;
    float2 l2 = make_float2(0.f, 0.f), e2 = l2;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
      unpack16<DT>(cur[u], x);
#pragma unroll
      for (int j = 0; j < N; j += 2) {
        float2 d = add2(make_float2(x[j], x[j + 1]), make_float2(-mm, -mm));
        d.x = max_nan(d.x, -1e5f);  // -inf: no weight, and no NaN from 0 * inf
        d.y = max_nan(d.y, -1e5f);
        const float2 z = mul2(d, make_float2(kLog2e, kLog2e));
        const float2 p = make_float2(ex2(z.x), ex2(z.y));
        l2 = add2(l2, p);
        e2 = fma2(d, p, e2);
      }
    }
    const float l = l2.x + l2.y;
    // e is relative to the maximum: a shift by d of all logits adds d l
    const float before = rest + last;
    e = (rise ? fmaf(-down, before, e) * f : e) - (e2.x + e2.y);
    rest = rise ? before * f : rest + l;
    last = rise ? l : last;
    held = rise ? b : held;
    m = nm;
  }

  // ---- maxima of 32 groups of 8 threads, and t ----
  float gm = m;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) gm = max_nan(gm, __shfl_xor_sync(0xffffffffu, gm, o));
  if ((lane & 7) == 0) sm.group_max[warp * 4 + (lane >> 3)] = gm;
  __syncthreads();
  float pm = -INFINITY, thr;
  {
    const float mine = sm.group_max[lane];
    int ahead = 0;
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 g4 = *reinterpret_cast<const float4*>(&sm.group_max[j]);
      const float g[4] = {g4.x, g4.y, g4.z, g4.w};
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        pm = max_nan(pm, g[y]);
        ahead += g[y] > mine || (g[y] == mine && j + y < lane);
      }
    }
    const unsigned who = __ballot_sync(0xffffffffu, ahead == max(a.top, 1) - 1);
    thr = __shfl_sync(0xffffffffu, mine, who ? __ffs(who) - 1 : 0);
  }
  const int lane_batches = (b1 - b0) * 32;
  if (thr == -INFINITY && a.top > 0 && lane_batches <= kLpFew) {
    // Fewer groups than `top` have logits, as in short rows: the top-th largest of the lane
    // batches' maxima.
    if (t == 0) sm.thr = -INFINITY;
    __syncthreads();
    for (int i = t; i < lane_batches; i += kLpThreads) {
      const float mine = maxima[i];
      int ahead = 0;
      for (int j = 0; j < lane_batches; ++j) ahead += maxima[j] > mine || (maxima[j] == mine && j < i);
      if (ahead == a.top - 1) sm.thr = mine;
    }
    __syncthreads();
    thr = sm.thr;
  }
  // pm: the piece's maximum; -inf where it has none, NaN where the row has no distribution
  const bool plain = pm > -INFINITY && pm < INFINITY;
  const bool ordered = pm == pm;  // no NaN

  // ---- the lane batches that reach t ----
  if (ordered && thr > -INFINITY && a.top > 0) {
    for (int i = t; i < lane_batches; i += kLpThreads)
      if (maxima[i] >= thr) {
        const int at = atomicAdd(&sm.listed, 1);
        if (at < kLpList) sm.list[at] = i;
      }
  }
  __syncthreads();
  const int listed = min(sm.listed, kLpList);
  const bool all_listed = ordered && thr > -INFINITY && sm.listed <= kLpList;
  // Threads of the maximum leave out the batch it came from: it is summed again without it.
  const bool top_thread = m == pm;
  float l = 0.f, pe = 0.f;
  int n = 0;
  if (held >= 0 && plain) {
    const float d = max_nan(m - pm, -1e5f), f = ex2(d * kLog2e);
    l = top_thread ? rest : (rest + last) * f;
    pe = (top_thread ? e : fmaf(-d, rest + last, e)) * f;
    if (m == -INFINITY) l = pe = 0.f;
  }
  if (top_thread && held >= 0 && plain) {
#pragma unroll 1
    for (int u = 0; u < U; ++u) {
      float x[N];
      unpack16<DT>(load1(held * 32 * U + lane + 32 * u), x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (x[j] == pm)
          ++n;
        else
          l += ex2(max_nan(x[j] - pm, -1e5f) * kLog2e);
      }
    }
  }
  // The logits of the listed lane batches from `least` on (or above it): candidates.
  auto gather = [&](int n, float least, bool above) {
    for (int i = t; i < n * U; i += kLpThreads) {
      const int k = sm.list[i / U];  // vector i % U of lane batch k
      const int v = (b0 + k / 32) * 32 * U + k % 32 + 32 * (i % U);
      if (v >= vecs) continue;
      float x[N];
      unpack16<DT>(load1(v), x);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int idx = v * N + j - lead;
        if (x[j] >= least && !(above && x[j] == least) && idx >= 0 && idx < a.vocab) {
          const int at = atomicAdd(&sm.count, 1);
          if (at < kLpCand) sm.cand[at] = token_key(x[j], idx);
        }
      }
    }
  };
  if (a.top > 0 && all_listed) gather(listed, thr, false);
  l = warp_sum(l);
  pe = warp_sum(pe);
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) sm.red_l[warp] = l, sm.red_e[warp] = pe, sm.red_n[warp] = n;
  if (pieces > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  __syncthreads();
  if (t == 0) {
    float tl = 0.f, te = 0.f;
    int tn = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) tl += sm.red_l[w], te += sm.red_e[w], tn += sm.red_n[w];
    out->m = pm, out->l = tl, out->e = te, out->n = tn;
  }

  // Too many logits reach t, or t is -inf: those above t as candidates. Where they are too many
  // as well, t rises, by halving, to the top-th largest of the lane batches' maxima, so that fewer
  // than `top` lane batches have anything above it; and then to the top-th largest of those.
  auto few_above = [&] {
    for (int stage = 0;; ++stage) {
      __syncthreads();
      if (stage < 2) {
        if (t == 0) sm.listed = 0;
        __syncthreads();
        for (int i = t; i < lane_batches; i += kLpThreads)
          if (maxima[i] > thr) {
            const int at = atomicAdd(&sm.listed, 1);
            if (at < kLpList) sm.list[at] = i;
          }
      }
      if (t == 0) sm.count = 0;
      __syncthreads();
      const int n = sm.listed;
      if (n <= kLpList) {
        gather(n, thr, true);
        __syncthreads();
        if (sm.count <= kLpCand) return;
      }
      uint32_t lo = order_of(thr), hi = order_of(pm) + 1;  // `top` or more reach lo, not hi
      while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const float least = value_of(mid);
        int reach = 0;
        if (stage == 0) {
          for (int i = t; i < lane_batches; i += kLpThreads) reach += maxima[i] >= least;
        } else {
          for (int i = t; i < n * U; i += kLpThreads) {
            const int k = sm.list[i / U];
            float x[N];
            unpack16<DT>(load1((b0 + k / 32) * 32 * U + k % 32 + 32 * (i % U)), x);
#pragma unroll
            for (int j = 0; j < N; ++j) reach += x[j] >= least;  // above t: in the row
          }
        }
        reach = __reduce_add_sync(0xffffffffu, reach);
        __syncthreads();
        if (lane == 0) sm.red_n[warp] = reach;
        __syncthreads();
        reach = 0;
        for (int w = 0; w < W; ++w) reach += sm.red_n[w];
        (reach >= a.top ? lo : hi) = mid;
      }
      thr = value_of(lo);
    }
  };
  // The places behind the candidates: the first logits that equal t, by one warp.
  auto fill = [&] {
    int at = sm.count;
    if (warp > 0) return;
    for (int b = b0; b < b1 && at < a.top; ++b) {
      const bool has = maxima[(b - b0) * 32 + lane] >= thr;
      if (!__any_sync(0xffffffffu, has)) continue;
#pragma unroll 1
      for (int u = 0; u < U; ++u) {
        const int v = b * 32 * U + lane + 32 * u;
        uint32_t equal = 0;  // a bit for each of the vector's values
        if (has) {
          float x[N];
          unpack16<DT>(load1(v), x);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const int idx = v * N + j - lead;
            if (x[j] == thr && idx >= 0 && idx < a.vocab) equal |= 1u << j;
          }
        }
        int mine = __popc(equal), upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += up;
        }
        for (int k = at + upto - mine; equal && k < a.top; ++k, equal &= equal - 1)
          out->keys[k] = token_key(thr, v * N + __ffs(equal) - 1 - lead);
        at += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
  };

  // ---- the piece's largest, in order ----
  if (a.top > 0) {
    auto place = [&] {
      const int count = sm.count;
      for (int i = t; i < count; i += kLpThreads) {
        const unsigned long long mine = sm.cand[i];
        int ahead = 0;
        for (int j = 0; j < count; ++j) ahead += sm.cand[j] > mine;
        if (ahead < a.top) out->keys[ahead] = mine;
      }
    };
    // at least `top` logits reach t, or all that the piece has; ordinary rows' way is laid out first
    // (1,500 bf16 rows 101.3 us, 102.2 without the hint)
    if (__builtin_expect(all_listed && sm.count <= kLpCand, 1)) {
      place();
    } else if (ordered) {
      few_above();
      place();
      fill();
    } else {
      // no order among the maxima (NaN): one pass for each place
      unsigned long long prev = ~0ull;
      for (int r = 0; r < a.top && prev; ++r) {
        unsigned long long best = 0;
        for (int v = b0 * 32 * U + t; v < min(vecs, b1 * 32 * U); v += kLpThreads) {
          float x[N];
          unpack16<DT>(load1(v), x);
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const int idx = v * N + j - lead;
            const unsigned long long key = token_key(x[j], idx);
            if (idx >= 0 && idx < a.vocab && key < prev && key > best) best = key;
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const unsigned long long ob = __shfl_xor_sync(0xffffffffu, best, o);
          best = ob > best ? ob : best;
        }
        if (lane == 0) sm.red_k[warp] = best;
        __syncthreads();
        for (int w = 0; w < W; ++w) best = sm.red_k[w] > best ? sm.red_k[w] : best;
        if (t == 0) out->keys[r] = best;
        prev = best;
        __syncthreads();
      }
    }
  }

  // ---- CTA 0 joins the pieces ----
  if (pieces > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  {
    float pm = -INFINITY, pl = 0.f, pe = 0.f;
    int pn = 0;
    if (lane < pieces) {
      const LpPiece& p = sm.piece[lane];
      pm = p.m, pl = p.l, pe = p.e, pn = p.n;
    }
    float M = pm;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, o));
    // sums relative to M: those of a lower maximum shrink, its own logits among them
    const float d = fmaxf(pm - M, -1e5f), f = ex2(d * kLog2e);
    const bool top_piece = pm == M;
    float L = top_piece ? pl : (pl + pn) * f;
    float E = top_piece ? pe : fmaf(-d, pl + pn, pe) * f;
    L = warp_sum(L);
    E = warp_sum(E);
    const int same = __reduce_add_sync(0xffffffffu, top_piece ? pn : 0);
    const float others = L + static_cast<float>(same - 1);
    const float ln = isfinite(M) ? log1pf(others) : NAN;
    if (t == 0) {
      if (a.logprob) a.logprob[row] = target >= 0 ? (target_x - M) - ln : 0.f;
      if (a.entropy) a.entropy[row] = ln + E / (1.0f + others);
    }
    if (a.top > 0) {
      // a key's place: how many of every piece's, which are in order, are ahead of it
      const int all = pieces * a.top;
      for (int i = t; i < all; i += kLpThreads) {
        const unsigned long long mine = sm.piece[i / a.top].keys[i % a.top];
        if (mine == 0) continue;
        int ahead = 0;
        for (int j = 0; j < pieces; ++j) {
          const unsigned long long* keys = sm.piece[j].keys;
          int n = 0;
#pragma unroll
          for (int h = kLpMaxTop / 2; h > 0; h >>= 1)
            if (keys[n + h - 1] > mine) n += h;
          ahead += n + (keys[n] > mine ? 1 : 0);
        }
        if (ahead < a.top) {
          a.top_ids[row * a.top + ahead] = static_cast<int>(key_index(mine));
          a.top_logprobs[row * a.top + ahead] = (key_value(mine) - M) - ln;
        }
      }
    }
  }
}

template <int DT, int U>
cudaError_t launch(const LogprobArgs& a, cudaStream_t s) {
  constexpr int N = Vec<DT>::kVals, kBatch = 32 * U * N, kWarps = kLpThreads / 32;
  const int batches = (a.vocab + N - 1 + kBatch - 1) / kBatch + 1;  // the row may start anywhere in a vector
  // As many pieces as the GPU's 148 SMs hold at once, and a piece's maxima fit (one float per
  // lane batch); none of less than a batch for each of its warps.
  constexpr int kSlots = 4;  // CTAs of an SM
  int pieces = 1;
  auto batches_each = [&] { return (batches + pieces - 1) / pieces; };
  // Clusters of more than 8 find room on an idle GPU only: 64 rows in 16 pieces take twice as long as in 8.
  const int most = a.rows <= 8 ? kLpMaxCluster : 8;
  while ((pieces < kLpMaxCluster && batches_each() > 320) ||
         (pieces < most && static_cast<long long>(a.rows) * (pieces + 1) <= kSlots * 148 &&
          batches >= (pieces + 1) * kWarps))
    ++pieces;
  const size_t smem = sizeof(LpShared) + static_cast<size_t>(batches_each()) * 32 * sizeof(float);
  static std::atomic<unsigned long long> configured{0};
  once_per_device(configured, [&] {
    cudaFuncSetAttribute(logprobs_kernel<DT, U>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024);
    cudaFuncSetAttribute(logprobs_kernel<DT, U>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  });
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * pieces);
  cfg.blockDim = dim3(kLpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pieces;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pieces > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, logprobs_kernel<DT, U>, a, batches_each());
}

// Short rows take one vector a lane, so that all lanes have some and the candidates are few.
template <int DT>
cudaError_t launch(const LogprobArgs& a, cudaStream_t s) {
  return a.vocab <= kLpThreads * 4 * Vec<DT>::kVals ? launch<DT, 1>(a, s) : launch<DT, 4>(a, s);
}

}  // namespace

cudaError_t op_token_logprobs(const LogprobArgs& a, cudaStream_t s) {
  return a.dtype == kDtBf16 ? launch<kDtBf16>(a, s) : launch<kDtF32>(a, s);
}

}  // namespace orx
