// Grouped-query attention of the last tokens of a batch of sequences over the
// 8-bit paged KV cache, with leading pages that all sequences share.
#include <cooperative_groups.h>

#include <algorithm>

#include "kv_quant.cuh"

namespace cg = cooperative_groups;

namespace orx {
using namespace kvq;
namespace {

// ---- attention --------------------------------------------------------------
// Per kv head, the query rows that read a page -- (query token, head of the
// group), and for shared pages those of every sequence -- are the columns of
//   S^T = K Q^T  (16 tokens x 8 columns, depth D)  and  O^T += V^T P^T,
// as mma.sync m16n8k16 with fp16 operands and fp32 sums: a decode step has a
// few columns only, and the cache's bytes bound it, not the products. Codes
// are exact in fp16. Scales stay outside: K's multiplies the score, V's the
// probability,  p_j = 2^(z_j - r),  l = sum p_j,  O = sum (p_j vs_j) c_j,
// and the reference r is what the products need: near the largest
// z_j + log2 vs_j, so that p_j vs_j stays in fp16's range whatever the V scales
// are, down to 2^-104 (fp32 holds p_j and l in between). A query row is scaled by a power of
// two to fp16's upper end; fp32 rows and their products are held as two fp16
// parts (22 bits), bf16 rows' queries are exact in one and their products
// rounded to one (2^-11). r only rises, and only when a score passes it by
// more than 2^4, so most pages need no reduction across lanes; sums of p are
// per lane until the end.
//
// A page's codes are turned to fp16 once for 8 columns, or once for 16 where a
// sequence has more than 8 query rows: 60 sequences of 64 rows 59 us and 66 with
// 8 columns, of 64 values 44 and 60; 200 of 16 rows and up to 9,000 tokens 74
// and 89. The two parts of fp32 rows of 128 values leave no registers for it
// (84 and 71); of 64 values 49 and 61. Of 64 values also where rows of several
// sequences share more pages than they may have of their own (260 fp32 rows a
// head behind 13,800 tokens 57 and 75 us; 24 bf16 rows of 128 values 35 and 31).
//
// Work: a job is (kv head, 8 or 16 columns, a run of pages): first the shared pages'
// jobs, then each sequence's own. All jobs' pages in one row are cut into
// equal shares, one per warp, whatever the lengths are -- a job begins with
// kStart units that are no pages, as beginning a piece takes a warp as long as
// some pages (64 sequences of 1 to 1,452 tokens 41.8 us with 0 of them, 32.6
// with 1, 28.9 with 3, 29.5 with 6) --; a share's part of a job is a piece. A job in one piece and without shared pages is finished at
// once; otherwise pieces leave (m, l, O) and kvq_join_kernel adds them in
// order.
constexpr int kWarps = 11;            // consumers per CTA, one CTA per SM; one more warp fetches for them
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kShares = kWarps * kCtas;
constexpr int kSlots = 4;             // blocks of a warp's ring
constexpr int kAhead = 4;             // page ids under way per warp
constexpr int kIds = 8;
constexpr int kCols = 8;
// The shared pages go to tcgen05 (kv_shared.cu) where more rows than this read
// them, and the warps here would get more than 4 pages of them each.
constexpr int kTcRows = 32;
constexpr long long kTcUnits = 4 * kShares;
constexpr unsigned kFewRows = 256, kManyRows = 1024;  // up to and from where the join gives a row 32 warps and one
constexpr int kStart = 3;             // what beginning a piece costs a warp, in pages
constexpr int kBins = kThreads;       // sequences are found through sums over up to this many runs of them
// What one (kv head, columns) job of n pages costs, in units of a page.
__device__ __forceinline__ int job_units(int n) { return n > 0 ? kStart + n : 0; }
// Sums of a job's units of the first `bin`, 2 `bin`, ... sequences in
// cum[1..kBins] (cum[0] = 0). All kBins threads of the CTA; ends with a barrier.
__device__ __forceinline__ void sum_units(const KvqCache& c, const KvqAttention& a, int bin,
                                          int* cum, int* tmp) {
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  int sum = 0;
  const long long b0 = static_cast<long long>(t) * bin;
  for (long long b = b0; b < b0 + bin && b < c.seqs; ++b) sum += job_units(own_pages(c, a, static_cast<int>(b)));
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) tmp[warp] = sum;
  __syncthreads();
  const int before = __reduce_add_sync(0xffffffffu, lane < warp ? tmp[lane] : 0);
  cum[t + 1] = before + sum;
  if (t == 0) cum[0] = 0;
  __syncthreads();
}

__device__ __forceinline__ void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2,
                                        uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Transposes an 8 x 8 matrix of fp16 held two per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
constexpr int kFirst = 1, kLast = 2;          // page of its piece
constexpr int kNoPage = 4;                    // outside the pool
constexpr int kJobStart = 8, kJobEnd = 16;    // of the last page: what of the job the piece has
constexpr int kShareEnd = 32, kNothing = 64;  // the share's last page; a share without any
struct alignas(16) PageTask {  // what a ring slot holds
  int page, flags;             // page: position / 16
  int job, head;
  int seq, col0;               // seq: -1 for shared pages
  int pad[2];
};

template <int D>
struct DecodeSmem {
  alignas(16) uint8_t ring[kWarps][kSlots][kvq_block_bytes(D)];
  PageTask task[kWarps][kSlots];
  uint64_t posted[kWarps][kSlots], full[kWarps][kSlots], empty[kWarps][kSlots];
  int ids[kWarps][kIds], seqs[kWarps][kIds];  // page ids under way, and whose
  int fail;  // a wait that ran out: the others do not wait either
  int cum[kBins + 1];
  int tmp[kWarps + 1];
};

// What a warp holds of a piece: 8 NT query rows of one kv head as columns, their
// references, sums and O.
template <int D, int FMT, int DT, int NT>
struct Piece {
  static constexpr bool kTwo = DT == kDtF32;  // two fp16 parts
  static constexpr int kW = D / 32;  // 4-code words of a V row in a lane; half of those of a K row
  int g, t;            // of the lane in the fragments
  uint32_t qh[NT][2 * kW][2], ql[NT][2 * kW][2];  // B fragments of Q^T: column g, the codes of chunk t (and t + 4)
  float o[NT][2 * kW][4];  // columns 2t, 2t + 1; value D / 8 * g + 2 i (+ 1) of MMA i
  float m[NT][2], l[NT][2], qf[NT][2];  // m: the reference r
  int limit[NT][2];    // keys that columns 2t, 2t + 1 (of the n-th 8) see
  int all_see, some_sees;  // keys that every column of the piece sees, and that any does
  int p_seq, head, col0, cols;

  __device__ __forceinline__ explicit Piece(int lane) : g(lane >> 2), t(lane & 3) {}

  // Columns [col, col + 8 NT) of kv head h, of sequence `seq` (-1: of all, at the shared pages).
  __device__ __forceinline__ void start(const KvqCache& c, const KvqAttention& a, const Plan& p,
                                        int seq, int h, int col) {
    p_seq = seq, head = h, col0 = col;
    cols = seq < 0 ? c.seqs * p.rows : p.rows;
    int least = 0x7fffffff, most = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int mycol = col0 + 8 * n + g;
      const bool live = mycol < cols;
      const Column cg = column_of(p, p_seq, live ? mycol : 0);
      const long long qrow = (static_cast<long long>(cg.seq) * a.q_tokens + cg.token) * a.q_stride +
                             static_cast<long long>(head * p.group + cg.head) * D;
      float q[2 * kW][4];
#pragma unroll
      for (int ch = 0; ch < kW / 2; ++ch)  // chunk t, then chunk t + 4
        load16<DT>(a.q, qrow + 16 * (t + 4 * ch), p.q_vec, q[4 * ch]);
      const int mine = live ? seq_len(c, a, cg.seq) - a.q_tokens + cg.token + 1 : 0;
      uint32_t amax = 0;
#pragma unroll
      for (int w = 0; w < 2 * kW; ++w) {
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (!live) q[w][x] = 0.f;
          amax = max(amax, __float_as_uint(q[w][x]) & 0x7fffffffu);
        }
      }
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      if (live) least = min(least, mine);
      most = max(most, mine);
      // 2^up brings the row's largest value to [2^14, 2^15); in two steps, as 2^up may be no number
      const int up = amax ? 14 - (static_cast<int>(amax >> 23) - 127) : 0;
      const float f1 = amax >= 0x7f800000u ? NAN : __uint_as_float((127 + up / 2) << 23);
      const float f2 = __uint_as_float((127 + up - up / 2) << 23);
#pragma unroll
      for (int w = 0; w < 2 * kW; ++w) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float y0 = q[w][2 * x] * f1 * f2, y1 = q[w][2 * x + 1] * f1 * f2;
          qh[n][w][x] = pack_half(y0, y1);
          if (kTwo) {
            const float2 h = unpack_half(qh[n][w][x]);
            ql[n][w][x] = pack_half(y0 - h.x, y1 - h.y);
          }
        }
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int down = -__shfl_sync(0xffffffffu, up, (2 * t + x) * 4);  // scores come out 2^up too large
        limit[n][x] = __shfl_sync(0xffffffffu, mine, (2 * t + x) * 4);
        qf[n][x] = a.scale * kLog2e * __uint_as_float((127 + down / 2) << 23) *
                   __uint_as_float((127 + down - down / 2) << 23);
        m[n][x] = -INFINITY;
        l[n][x] = 0.f;
      }
#pragma unroll
      for (int w = 0; w < 2 * kW; ++w) o[n][w][0] = o[n][w][1] = o[n][w][2] = o[n][w][3] = 0.f;
    }
    all_see = __reduce_min_sync(0xffffffffu, least);
    some_sees = __reduce_max_sync(0xffffffffu, most);
  }

  // NP pages from position / 16 = `page` on; `fine`: bit i, page i is there.
  template <int NP>
  __device__ __forceinline__ void step(const uint8_t* blk0, const uint8_t* blk1, int page, int fine) {
    const bool edge = (page + NP) * kPage > all_see || fine != (1 << NP) - 1;
    // ---- S^T, in independent sums ----
    float s[NT][2 * NP][2];  // [8 tokens][column 2t, 2t + 1]
#pragma unroll
    for (int y = 0; y < NP; ++y) {
      const uint8_t* blk = y ? blk1 : blk0;
      float sa[NT][kTwo ? 4 : 2][4] = {};
#pragma unroll
      for (int ch = 0; ch < D / 64; ++ch) {
        const uint4 r0 = *reinterpret_cast<const uint4*>(blk + g * D + 16 * (t + 4 * ch));
        const uint4 r1 = *reinterpret_cast<const uint4*>(blk + (g + 8) * D + 16 * (t + 4 * ch));
        const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t a0, a1, a2, a3;
          codes_to_half<FMT>(w0[w], a0, a2);
          codes_to_half<FMT>(w1[w], a1, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const auto& h = qh[n][4 * ch + w];
            mma_f16(sa[n][w & 1], a0, a1, a2, a3, h[0], h[1]);
            const auto& lo = ql[n][4 * ch + w];
            if (kTwo) mma_f16(sa[n][2 + (w & 1)], a0, a1, a2, a3, lo[0], lo[1]);
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          s[n][2 * y + k / 2][k & 1] =
              kTwo ? (sa[n][0][k] + sa[n][1][k]) + (sa[n][kTwo ? 2 : 0][k] + sa[n][kTwo ? 3 : 0][k])
                   : sa[n][0][k] + sa[n][1][k];
    }
    // ---- probabilities of tokens g + 8 y in columns 2t, 2t + 1 ----
    float ks[2 * NP], vs[2 * NP], e[2 * NP];
#pragma unroll
    for (int y = 0; y < 2 * NP; ++y) {
      const float* sc = reinterpret_cast<const float*>((y < 2 ? blk0 : blk1) + 2 * kPage * D);
      ks[y] = sc[g + 8 * (y & 1)];
      vs[y] = sc[kPage + g + 8 * (y & 1)];
      e[y] = scale_exponent(vs[y]);
    }
    uint32_t pb[NT][2 * NP], pl[NT][2 * NP];  // B fragments of P^T, and its second parts
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float z[2 * NP][2], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int y = 0; y < 2 * NP; ++y) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          z[y][x] = s[n][y][x] * (qf[n][x] * ks[y]);
          if (edge && !(page * kPage + g + 8 * y < limit[n][x] && (fine >> (y >> 1) & 1)))
            z[y][x] = -INFINITY;
          top[x] = fmaxf(top[x], z[y][x] + e[y]);
        }
      }
      if (__any_sync(0xffffffffu, top[0] > m[n][0] + kSlack || top[1] > m[n][1] + kSlack)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1)
            top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], d));
          // each column by its own scores alone, whatever rows share its tile
          if (top[x] > m[n][x] + kSlack) {
            const float h = ex2_half(m[n][x] - top[x]), f = h * h;
            m[n][x] = top[x];
            l[n][x] = l[n][x] * h * h;
#pragma unroll
            for (int w = 0; w < 2 * kW; ++w) {
              o[n][w][x] *= f;
              o[n][w][2 + x] *= f;
            }
          }
        }
      }
      const float mk[2] = {m[n][0] - kLift, m[n][1] - kLift};
#pragma unroll
      for (int y = 0; y < 2 * NP; ++y) {
        float pv[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const bool none = edge && z[y][x] == -INFINITY;
          const float pr = none ? 0.f : ex2(z[y][x] - mk[x]);
          l[n][x] += pr;
          pv[x] = none ? 0.f : pr * vs[y];
        }
        const uint32_t h = pack_half(pv[0], pv[1]);
        pb[n][y] = transpose8(h);
        if (kTwo) {
          const float2 f = unpack_half(h);
          pl[n][y] = transpose8(pack_half(pv[0] - f.x, pv[1] - f.y));
        }
      }
    }
    // ---- O^T += V^T P^T: tokens 2t, 2t + 1, 2t + 8, 2t + 9, values D / 8 * g ... ----
#pragma unroll
    for (int y = 0; y < NP; ++y) {
      const uint8_t* blk = y ? blk1 : blk0;
      uint32_t vw[4][kW];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int tok = 2 * t + (k & 1) + (k >> 1) * 8;
        const uint8_t* src = blk + (kPage + tok) * D + D / 8 * g;
        if (D == 128) {
          const uint4 r = *reinterpret_cast<const uint4*>(src);
          vw[k][0] = r.x, vw[k][1] = r.y, vw[k][kW - 2] = r.z, vw[k][kW - 1] = r.w;
        } else {
          const uint2 r = *reinterpret_cast<const uint2*>(src);
          vw[k][0] = r.x, vw[k][1] = r.y;
        }
        if (FMT == kKvqE4m3 && edge &&
            !((page + y) * kPage + tok < some_sees && (fine >> y & 1))) {
          // never written, perhaps the code of a NaN, which 0 * would keep
#pragma unroll
          for (int w = 0; w < kW; ++w) vw[k][w] = 0;
        }
      }
#pragma unroll
      for (int w = 0; w < kW; ++w) {
#pragma unroll
        for (int hw = 0; hw < 2; ++hw) {  // codes 0, 1 and 2, 3 of the word
          const int sel = hw ? 0x7362 : 0x5140;
          uint32_t a0, a1, a2, a3;
          codes_to_half<FMT>(__byte_perm(vw[0][w], vw[1][w], sel), a0, a1);
          codes_to_half<FMT>(__byte_perm(vw[2][w], vw[3][w], sel), a2, a3);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_f16(o[n][2 * w + hw], a0, a1, a2, a3, pb[n][2 * y], pb[n][2 * y + 1]);
            if (kTwo) mma_f16(o[n][2 * w + hw], a0, a1, a2, a3, pl[n][2 * y], pl[n][2 * y + 1]);
          }
        }
      }
    }
  }

  // From here on pages of sequence b alone: the other columns see none of them.
  __device__ __forceinline__ void only(const Plan& p, int b, const int (&full)[NT][2]) {
    int most = 0;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        limit[n][x] = p.by_rows.of(col0 + 8 * n + 2 * t + x) == b ? full[n][x] : 0;
        most = max(most, limit[n][x]);
      }
    all_see = 0;
    some_sees = __reduce_max_sync(0xffffffffu, most);
  }

  // The lanes' sums together; r and l are then the piece's.
  __device__ __forceinline__ void close() {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[n][x] += __shfl_xor_sync(0xffffffffu, l[n][x], d);
  }
  // Column 8n + 2t + x's record (D values, r, l) at rec, by its 8 lanes.
  __device__ __forceinline__ void put(int n, int x, float* rec) const {
#pragma unroll
    for (int w = 0; w < kW; ++w)
      *reinterpret_cast<float4*>(rec + D / 8 * g + 4 * w) =
          make_float4(o[n][2 * w][x], o[n][2 * w][2 + x], o[n][2 * w + 1][x], o[n][2 * w + 1][2 + x]);
    if (g == 0) *reinterpret_cast<float2*>(rec + D) = make_float2(m[n][x] - kLift, l[n][x]);
  }
};

// Two records as one: a += b.
template <int E>
__device__ __forceinline__ void join_into(float& m, float& l, float* o, float bm, float bl,
                                          const float* bo) {
  if (bl == 0.f) return;
  const float nm = fmaxf(m, bm), h = ex2_half(m - nm), bh = ex2_half(bm - nm), f = h * h, bf = bh * bh;
  l = l * h * h + bl * bh * bh;
#pragma unroll
  for (int x = 0; x < E; ++x) o[x] = o[x] * f + bo[x] * bf;
  m = nm;
}
// A warp's D values of a record, E = D / 32 a lane.
template <int E>
__device__ __forceinline__ void load_lane(const float* p, float* v) {
  if (E == 4) {
    const float4 w = *reinterpret_cast<const float4*>(p);
    v[0] = w.x, v[1] = w.y, v[E - 2] = w.z, v[E - 1] = w.w;
  } else {
    const float2 w = *reinterpret_cast<const float2*>(p);
    v[0] = w.x, v[1] = w.y;
  }
}
// Row `row`, query head h: the finished output of a warp's record.
template <int D, int DT>
__device__ __forceinline__ void put_row(const KvqAttention& a, const Plan& p, int row, int h, int lane,
                                        float m, float l, const float* o) {
  constexpr int E = D / 32;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const long long at = static_cast<long long>(row) * a.out_stride + h * D + lane * E;
  if (p.out_vec && DT == kDtBf16) {
#pragma unroll
    for (int x = 0; x < E; x += 2)
      reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at)[x / 2] =
          pack_bf16(o[x] * inv, o[x + 1] * inv);
  } else {
#pragma unroll
    for (int x = 0; x < E; ++x) store_f(a.out, DT, at + x, o[x] * inv);
  }
  if (lane == 0 && a.lse)
    a.lse[static_cast<long long>(row) * a.q_heads + h] = l == 0.f ? -INFINITY : ln_sum(m, l);
}

// Pages in the order of the shares: sequence (-1: the shared pages) and its
// job, page in [.., end); `left` units of the share, 0 or less behind its last
// page.
struct Cursor {
  int seq, job, page, end, left;
  // find(seq): the next sequence that has pages; called if there is one.
  template <typename F>
  __device__ __forceinline__ void next(const KvqCache& c, const KvqAttention& a, const Plan& p,
                                       int seq_jobs, F&& find) {
    --left;
    if (++page < end) return;
    left -= kStart;
    if (left <= 0) return;
    page = seq < 0 ? 0 : a.shared_pages;
    if (++job < (seq < 0 ? p.shared_jobs : seq_jobs)) return;
    job = 0;
    seq = find(seq);
    page = a.shared_pages;
    end = page + own_pages(c, a, seq);
  }
};

// The fetching warp: lane w keeps consumer warp w's ring full with the pages of
// its share, in order, and describes each in its slot's task. Page ids come
// kAhead pages before they are used, without a stall, by asynchronous copies.
template <int D>
__device__ void fetch_pages(const KvqCache& c, const KvqAttention& a, const Plan& p,
                            DecodeSmem<D>& sm, long long units, int lane) {
  constexpr int kBlk = kvq_block_bytes(D);
  const Share share = share_of(blockIdx.x * kWarps + lane, units, kShares);
  const bool mine = lane < kWarps && share.count > 0;
  const unsigned lanes = __ballot_sync(0xffffffffu, mine);
  if (!mine) return;
  const int seq_jobs = c.kv_heads * p.tiles;
  Cursor at;
  if (share.start < p.shared_units) {
    at.seq = -1;
    at.job = static_cast<int>(share.start / (kStart + a.shared_pages));
    at.page = static_cast<int>(share.start - static_cast<long long>(at.job) * (kStart + a.shared_pages));
    at.end = a.shared_pages;
  } else {
    const long long v = share.start - p.shared_units;
    int lo = 0, hi = kBins;  // largest bin whose sum before it is <= v
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (static_cast<long long>(sm.cum[mid]) * seq_jobs <= v)
        lo = mid;
      else
        hi = mid;
    }
    long long rest = v - static_cast<long long>(sm.cum[lo]) * seq_jobs;
    at.seq = lo * p.bin;
    int n = p.bin == 1 ? sm.cum[lo + 1] - sm.cum[lo] : job_units(own_pages(c, a, at.seq));
    while (rest >= static_cast<long long>(n) * seq_jobs) {
      rest -= static_cast<long long>(n) * seq_jobs;
      n = job_units(own_pages(c, a, ++at.seq));
    }
    at.job = static_cast<int>(rest <= 0xffffffffll ? static_cast<uint32_t>(rest) / static_cast<uint32_t>(n)
                                                   : rest / n);
    at.page = a.shared_pages + static_cast<int>(rest - static_cast<long long>(at.job) * n);
    at.end = a.shared_pages + n - kStart;
  }
  // at.page is now the place among the job's units, of which the first kStart are no pages
  const int first = at.seq < 0 ? 0 : a.shared_pages, over = at.page - first - kStart;
  at.page = first + max(over, 0);
  at.left = share.count + min(over, 0);
  if (at.left <= 0) {
    sm.task[lane][0].flags = kNothing;
    mbar_arrive(&sm.posted[lane][0]);
  }
  Cursor ahead = at;
  int asked = 0;
  // Behind seq. Whole runs of empty sequences are passed by their sums (8,000 sequences, 64 at the
  // ends with 1,000 tokens, 99 us; one by one 995).
  auto find = [&](int seq) {
    while (own_pages(c, a, ++seq) == 0 && seq + 1 < c.seqs) {
      int bin = (seq + 1) / p.bin;
      if (seq + 1 != bin * p.bin) continue;
      while (bin + 1 < kBins && sm.cum[bin + 1] == sm.cum[bin]) ++bin;
      seq = min(bin * p.bin, c.seqs - 1) - 1;
    }
    return seq;
  };
  auto ask = [&] {  // for the page id under `ahead`
    if (ahead.left > 0) {
      const int* src = ahead.seq < 0
                           ? a.shared + ahead.page
                           : c.page_table + static_cast<long long>(ahead.seq) * c.max_pages + ahead.page;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(
                       smem_u32(&sm.ids[lane][asked % kIds])),
                   "l"(src)
                   : "memory");
      sm.seqs[lane][asked % kIds] = ahead.seq;
      ++asked;
      ahead.next(c, a, p, seq_jobs, find);
    }
  };
  for (int i = 0; i < kAhead; ++i) ask();
  asm volatile("cp.async.commit_group;" ::: "memory");
  int tiles = at.seq < 0 ? p.shared_tiles : p.tiles;
  int head = at.job / tiles, tile = at.job - head * tiles;
  int piece = kFirst | (at.page == first ? kJobStart : 0);
  int slot = 0, phase = 1, fresh = 0;
  unsigned long long since = 0;
  for (int sent = 0; __any_sync(lanes, at.left > 0);) {
    // lanes whose ring is full go round again, while the others send
    const bool room = at.left > 0 && (sent < kSlots || mbar_test(&sm.empty[lane][slot], phase));
    if (!__any_sync(lanes, room)) {
      const unsigned long long now = global_ns();
      if (since == 0) since = now;
      if (now - since > kWaitLimitNs) {
        atomicExch(&sm.fail, kErrWaitTimeout);
        at.left = 0;
      }
      __nanosleep(20);
      continue;
    }
    since = 0;
    // an id was asked for at least kAhead - 1 of a lane's turns ago, each in a round of its own
    if (fresh < kAhead) {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      ++fresh;
    } else {
      asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    }
    if (room) {
      const int id = sm.ids[lane][sent % kIds];
      const bool job_end = at.page + 1 == at.end;
      const bool last = job_end || at.left == 1, end = at.left <= (job_end ? 1 + kStart : 1);
      const bool fine = id >= 0 && id < c.pages;
      PageTask& k = sm.task[lane][slot];
      const int flags = piece | (last ? kLast : 0) | (job_end ? kJobEnd : 0) | (end ? kShareEnd : 0) |
                        (fine ? 0 : kNoPage);
      const int job = at.seq < 0 ? at.job : p.shared_jobs + at.seq * seq_jobs + at.job;
      *reinterpret_cast<int4*>(&k) = make_int4(at.page, flags, job, head);
      *reinterpret_cast<int2*>(&k.seq) = make_int2(at.seq, tile * p.cols);
      mbar_arrive(&sm.posted[lane][slot]);
      uint64_t* bar = &sm.full[lane][slot];
      if (fine) {
        mbar_arrive_expect_tx(bar, kBlk);
        bulk_g2s(sm.ring[lane][slot],
                 c.pool + (static_cast<long long>(id) * c.kv_heads + head) * kBlk, kBlk, bar);
      } else {
        note_bad(c.err);
        mbar_arrive(bar);
      }
      piece &= ~kFirst;
      if (++slot == kSlots) slot = 0, phase ^= 1;
      ++sent;
      const int seq = at.seq;
      at.next(c, a, p, seq_jobs, [&](int) { return sm.seqs[lane][sent % kIds]; });  // asked for already
      if (at.left > 0) {
        if (job_end) {
          piece = kFirst | kJobStart;
          if (++tile == tiles) tile = 0, ++head;
          if (at.seq != seq) tile = head = 0, tiles = p.tiles;
        }
      }
      ask();
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
}

template <int D, int FMT, int DT, int NT>
__global__ void __launch_bounds__(kThreads, 1)
    kvq_decode_kernel(KvqCache c, KvqAttention a, Plan p) {
  constexpr int kW = D / 32;
  extern __shared__ __align__(16) uint8_t kvq_raw[];
  DecodeSmem<D>& sm = *reinterpret_cast<DecodeSmem<D>*>(kvq_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (threadIdx.x == 0) sm.fail = 0;
  if (warp < kWarps && lane == 0) {
    for (int i = 0; i < kSlots; ++i) {
      mbar_init(&sm.posted[warp][i], 1);
      mbar_init(&sm.full[warp][i], 1);
      mbar_init(&sm.empty[warp][i], 1);
    }
    fence_mbar_init();
  }
  pdl_trigger();  // every CTA runs from the start; the join waits for their ends
  sum_units(c, a, p.bin, sm.cum, sm.tmp);
  const long long units =
      p.shared_units + static_cast<long long>(sm.cum[kBins]) * c.kv_heads * p.tiles;
  if (warp == kWarps) {
    fetch_pages<D>(c, a, p, sm, units, lane);
    settle(&sm.fail);
    pdl_wait();
    return;
  }
  const int share = blockIdx.x * kWarps + warp;
  if (share_of(share, units, kShares).count == 0) {
    pdl_wait();
    return;
  }

  // Two pages a step; with int8's conversions, 16 columns of 128 values leave registers for one
  // (200 sequences, 12 rows: 31.6 us, 35.0 with the spills of two).
  constexpr bool kPairs = NT == 1 || D == 64 || FMT == kKvqE4m3;
  Piece<D, FMT, DT, NT> k(lane);
  int slot = 0, phase = 0;
  for (bool more = true; more;) {
    // without a task there is nothing to go by
    if (!__all_sync(0xffffffffu, mbar_sleep(&sm.posted[warp][slot], phase, &sm.fail))) break;
    const int4 first = *reinterpret_cast<const int4*>(&sm.task[warp][slot]);  // page, flags, job, head
    if (first.y & kNothing) break;
    if (first.y & kFirst) {
      // a new piece: its queries come while its first pages are on their way
      k.start(c, a, p, sm.task[warp][slot].seq, first.w, sm.task[warp][slot].col0);
    }
    const bool here = mbar_sleep(&sm.full[warp][slot], phase, &sm.fail);
    const int slot0 = slot, fine0 = here && !(first.y & kNoPage);
    if (++slot == kSlots) slot = 0, phase ^= 1;
    int4 task = first;
    if (!kPairs || (first.y & kLast)) {
      k.template step<1>(sm.ring[warp][slot0], nullptr, first.x, fine0);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.empty[warp][slot0]);
    } else {
      const bool here1 = mbar_sleep(&sm.full[warp][slot], phase, &sm.fail);
      task = *reinterpret_cast<const int4*>(&sm.task[warp][slot]);
      const int fine1 = here1 && !(task.y & kNoPage);
      k.template step<2>(sm.ring[warp][slot0], sm.ring[warp][slot], first.x, fine0 | fine1 << 1);
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.empty[warp][slot0]);
        mbar_arrive(&sm.empty[warp][slot]);
      }
      if (++slot == kSlots) slot = 0, phase ^= 1;
    }
    if (!(task.y & kLast)) continue;

    // ---- the piece is done ----
    more = !(task.y & kShareEnd);
    const bool finish = !p.joined && (task.y & kJobStart) && (task.y & kJobEnd);
    k.close();
#pragma unroll
    for (int nx = 0; nx < 2 * NT; ++nx) {
      const int n = nx / 2, x = nx % 2, col = k.col0 + 8 * n + 2 * t + x;
      if (col >= k.cols) continue;
      if (finish) {
        const Column cc = column_of(p, k.p_seq, col);
        const long long row = static_cast<long long>(cc.seq) * a.q_tokens + cc.token;
        const int h = k.head * p.group + cc.head;
        const float inv = k.l[n][x] == 0.f ? 0.f : 1.0f / k.l[n][x];
        const long long at = row * a.out_stride + static_cast<long long>(h) * D + D / 8 * g;
        float v[4 * kW];
#pragma unroll
        for (int w = 0; w < 2 * kW; ++w)
          v[2 * w] = k.o[n][w][x] * inv, v[2 * w + 1] = k.o[n][w][2 + x] * inv;
        if (p.out_vec) {
#pragma unroll
          for (int w = 0; w < 4 * kW; w += Wide<DT>::kVals) {
            if (DT == kDtBf16)
              *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + at + w) =
                  make_uint4(pack_bf16(v[w], v[w + 1]), pack_bf16(v[w + 2], v[w + 3]),
                             pack_bf16(v[w + 4], v[w + 5]), pack_bf16(v[w + 6], v[w + 7]));
            else
              *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at + w) =
                  make_float4(v[w], v[w + 1], v[w + 2], v[w + 3]);
          }
        } else {
#pragma unroll
          for (int w = 0; w < 4 * kW; ++w) store_f(a.out, DT, at + w, v[w]);
        }
        if (g == 0 && a.lse)
          a.lse[row * a.q_heads + h] = k.l[n][x] == 0.f ? -INFINITY : ln_sum(k.m[n][x] - kLift, k.l[n][x]);
      } else {
        k.put(n, x, p.records(a.ws) + (static_cast<long long>(share + task.z) * (8 * NT) + 8 * n +
                                       2 * t + x) * (D + 4));
      }
    }
    if (lane == 0) {
      int* dir = p.directory(a.ws) + 2 * task.z;
      if (task.y & kJobStart) dir[0] = share;
      if (task.y & kJobEnd) dir[1] = share;
    }
  }
  if (lane == 0 && c.err && *static_cast<volatile int*>(&sm.fail)) atomicExch(c.err, sm.fail);
  settle(&sm.fail);
  // the join, which waits for this kernel, needs the shared pages' too
  pdl_wait();
}

// The pieces of a query row and head: those of the shared pages, then its own.
struct RowPieces {
  const float *rec0, *rec1;  // the first of either
  int n0, n1;
  int row0;                  // place of the row in rec0's
  bool join;                 // false: finished by its one piece, or not there
};
template <int D>
__device__ __forceinline__ RowPieces row_pieces(const KvqCache& c, const KvqAttention& a, const Plan& p,
                                                unsigned r, bool there) {
  const int row = p.by_heads.of(r), h = r - row * a.q_heads;
  const int b = there ? p.by_tokens.of(row) : 0, tok = row - b * a.q_tokens;
  const int head = p.by_group.of(h), local = tok * p.group + h - head * p.group;
  const int n = own_pages(c, a, b);
  const int ccol = b * p.rows + local;
  const bool tc = p.tc_jobs > 0;
  const int width = tc ? kRows : p.cols;
  const int job0 = tc ? head * p.tc_tiles + ccol / kRows : head * p.shared_tiles + ccol / p.cols;
  const int job1 = p.shared_jobs + (b * c.kv_heads + head) * p.tiles + local / p.cols;
  if (there && local == 0 && a.lens[b] < 0) note_bad(c.err);  // no piece saw it
  pdl_wait();
  const int* dir = p.directory(a.ws);
  int2 d0 = make_int2(0, -1), d1 = d0;
  if (there && p.joined)
    d0 = *reinterpret_cast<const int2*>(dir + 2 * (tc ? p.jobs + job0 : job0));
  if (there && n > 0) d1 = *reinterpret_cast<const int2*>(dir + 2 * job1);
  RowPieces x;
  x.join = there && (p.joined || n == 0 || d1.x != d1.y);
  // shares that gave up (their error is noted) leave what was there before
  auto known = [](int2 d, int n) { return d.x >= 0 && d.x <= d.y && d.y < n; };
  if (p.joined && !known(d0, tc ? kCtas : p.shares)) x.join = false;
  if (n > 0 && !known(d1, p.shares)) x.join = false;
  x.n0 = d0.y - d0.x + 1, x.n1 = d1.y - d1.x + 1;
  x.row0 = ccol % width;
  x.rec0 = (tc ? p.tc_records(a.ws, D) : p.records(a.ws)) +
           static_cast<long long>(d0.x + job0) * width * (D + 4);
  x.rec1 = p.records(a.ws) + (static_cast<long long>(d1.x + job1) * p.cols + local % p.cols) * (D + 4);
  return x;
}
// A warp adds every kSplit-th piece from the part-th on, four at a time, in order.
template <int D, int kSplit>
__device__ __forceinline__ void add_pieces(const Plan& p, const RowPieces& x, int part, int lane, float& m,
                                           float& l, float* o) {
  constexpr int E = D / 32, kAt = 4;
  const bool tc = p.tc_jobs > 0;
  const int width = tc ? kRows : p.cols, all = x.n0 + x.n1, at = lane * E;
  const int ml0 = tc ? kRows * D + 2 * x.row0 : x.row0 * (D + 4) + D;
  const int val0 = tc ? at / 8 * (kRows * 8) + x.row0 * 8 + at % 8 : x.row0 * (D + 4) + at;
  m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  for (int i = part; i < all; i += kSplit * kAt) {
    float v[kAt][E];
    float2 ml[kAt];
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const int j = i + k * kSplit;
      ml[k] = make_float2(-INFINITY, 0.f);
      if (j < all) {
        const float* rec = j < x.n0 ? x.rec0 + static_cast<long long>(j) * width * (D + 4)
                                    : x.rec1 + static_cast<long long>(j - x.n0) * p.cols * (D + 4);
        ml[k] = *reinterpret_cast<const float2*>(rec + (j < x.n0 ? ml0 : D));
        load_lane<E>(rec + (j < x.n0 ? val0 : at), v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < kAt; ++k) join_into<E>(m, l, o, ml[k].x, ml[k].y, v[k]);
  }
}

// Adds the pieces of the query rows: kSplit warps a row where there are few
// rows, which may have a piece from every share (128 rows of 102 pieces: the
// whole call 48.3 us with 8 warps, 45.4 with 32), or a warp for `each` rows,
// whose lanes look up a row each, as most may be finished already (95,744 rows
// of one piece: the whole call 52 us with a warp for each, 30 with one for 21;
// 4,096 rows of 7 pieces: the join 27 us with eight warps a row, 12.5 with one).
constexpr int kJoinWarps = 8;
constexpr unsigned kJoinRows = kCtas * 32;  // rows from which on a warp has several
template <int D, int DT, int kSplit, bool kMany = false>  // kMany: `each` may be more than 1
__global__ void __launch_bounds__(kSplit > kJoinWarps ? 1024 : kJoinWarps * 32)
    kvq_join_kernel(KvqCache c, KvqAttention a, Plan p, int each) {
  constexpr int E = D / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rows = static_cast<unsigned>(c.seqs) * a.q_tokens * a.q_heads;
  float m, l, o[E];
  if constexpr (kSplit == 1 && !kMany) {
    const unsigned r = blockIdx.x * kJoinWarps + warp;
    const RowPieces x = row_pieces<D>(c, a, p, r, r < rows);
    if (!x.join) return;
    add_pieces<D, 1>(p, x, 0, lane, m, l, o);
    const int row = p.by_heads.of(r);
    put_row<D, DT>(a, p, row, r - row * a.q_heads, lane, m, l, o);
  } else if constexpr (kSplit == 1) {
    const unsigned first = (blockIdx.x * kJoinWarps + warp) * each;
    const RowPieces mine = row_pieces<D>(c, a, p, first + lane, lane < each && first + lane < rows);
    for (unsigned left = __ballot_sync(0xffffffffu, mine.join); left; left &= left - 1) {
      const int i = __ffs(left) - 1;
      RowPieces x;
      x.rec0 = reinterpret_cast<const float*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine.rec0), i));
      x.rec1 = reinterpret_cast<const float*>(
          __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine.rec1), i));
      x.n0 = __shfl_sync(0xffffffffu, mine.n0, i), x.n1 = __shfl_sync(0xffffffffu, mine.n1, i);
      x.row0 = __shfl_sync(0xffffffffu, mine.row0, i);
      add_pieces<D, 1>(p, x, 0, lane, m, l, o);
      const int row = p.by_heads.of(first + i);
      put_row<D, DT>(a, p, row, first + i - row * a.q_heads, lane, m, l, o);
    }
  } else {
    __shared__ float sh_o[kSplit][D], sh_m[kSplit], sh_l[kSplit];
    const unsigned r = blockIdx.x;
    const RowPieces x = row_pieces<D>(c, a, p, r, true);
    if (!x.join) return;
    add_pieces<D, kSplit>(p, x, warp, lane, m, l, o);
#pragma unroll
    for (int y = 0; y < E; ++y) sh_o[warp][lane * E + y] = o[y];
    if (lane == 0) sh_m[warp] = m, sh_l[warp] = l;
    __syncthreads();
    if (warp) return;
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < kSplit; ++w) m = fmaxf(m, sh_m[w]);
#pragma unroll
    for (int y = 0; y < E; ++y) o[y] = 0.f;
#pragma unroll
    for (int w = 0; w < kSplit; ++w) {
      if (sh_l[w] == 0.f) continue;
      const float h = ex2_half(sh_m[w] - m), f = h * h;
      l += sh_l[w] * h * h;
#pragma unroll
      for (int y = 0; y < E; ++y) o[y] += sh_o[w][lane * E + y] * f;
    }
    const int row = p.by_heads.of(r);
    put_row<D, DT>(a, p, row, r - row * a.q_heads, lane, m, l, o);
  }
}

// ---- short calls: one launch, a cluster of CTAs a job ----
// Where the sequences are short, or there is one, every job gets a cluster of
// its own, whose warps take equal runs of its pages, fetch them themselves and
// join through (distributed) shared memory: no workspace, no second launch. A
// job is (sequence, kv head, 8 rows); with shared pages (kv head, 8 rows of
// several sequences): the shared pages for all of them, and then the own pages
// of each, at which only its columns see anything.
constexpr int kJobWarps = 4, kJobSlots = 4;
template <int D>
struct JobSmem {
  alignas(16) uint8_t ring[kJobWarps][kJobSlots][kvq_block_bytes(D)];  // then each warp's records
  alignas(16) float rec[kCols][D + 4];                                 // the CTA's
  uint64_t full[kJobWarps][kJobSlots];
  int2 task[kJobWarps][kJobSlots];  // sequence (-1: shared) and page of a slot; page -1: not there
  int fail;
};
static_assert(kJobSlots * kvq_block_bytes(64) >= kCols * (64 + 4) * 4 &&
                  kJobSlots * kvq_block_bytes(128) >= kCols * (128 + 4) * 4,
              "a warp's records fit in its ring");

template <int D, int FMT, int DT>
__global__ void __launch_bounds__(kJobWarps * 32, 3)
    kvq_job_kernel(KvqCache c, KvqAttention a, Plan p) {
  constexpr int kBlk = kvq_block_bytes(D), E = D / 32;
  extern __shared__ __align__(16) uint8_t kvq_raw[];
  JobSmem<D>& sm = *reinterpret_cast<JobSmem<D>*>(kvq_raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int job = blockIdx.x / ctas;
  int b = -1, head, tile;  // b: the job's sequence, -1 where it has several
  if (p.joined) {
    head = job / p.group_tiles;
    tile = job - head * p.group_tiles;
  } else {
    const int seq_jobs = c.kv_heads * p.job_tiles;
    b = job / seq_jobs;
    head = (job - b * seq_jobs) / p.job_tiles;
    tile = job - b * seq_jobs - head * p.job_tiles;
  }
  if (lane == 0) {
    for (int i = 0; i < kJobSlots; ++i) mbar_init(&sm.full[warp][i], 1);
    fence_mbar_init();
  }
  if (threadIdx.x == 0) sm.fail = 0;
  __syncthreads();
  // The job's pages: `shared` shared ones, then those of sequences first + 0, 1, ... 7, whose last
  // ends at `ends` of lane 0, 1, ... 7.
  const int first = p.joined ? tile * kCols / p.rows : b;
  int shared = 0, ends = 0;
  {
    const int last = p.joined ? min(c.seqs, ((tile + 1) * kCols + p.rows - 1) / p.rows) : b + 1;
    int n = 0;
    if (first + lane < last) n = (seq_len(c, a, first + lane) + kPage - 1) / kPage;
    shared = min(p.joined ? a.shared_pages : 0, __reduce_max_sync(0xffffffffu, n));
    ends = p.joined ? max(0, n - a.shared_pages) : n;
#pragma unroll
    for (int o = 1; o < kCols; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, ends, o);
      if (lane >= o) ends += up;
    }
  }
  const int pages = shared + __shfl_sync(0xffffffffu, ends, kCols - 1);
  const Share share = share_of(rank * kJobWarps + warp, pages, ctas * kJobWarps);
  const int u0 = static_cast<int>(share.start), todo = share.count;
  // what the lane's page of a batch of 32 is: sequence, page and its place in the pool
  int now_b = -1, now_page = 0, now_id = -1, then_b = -1, then_page = 0, then_id = -1;
  auto look = [&](int k) {
    now_b = then_b, now_page = then_page, now_id = then_id;
    const int u = u0 + k + lane;
    int i = 0, before = 0;
#pragma unroll
    for (int x = 0; x < kCols; ++x) {
      const int e = __shfl_sync(0xffffffffu, ends, x);
      if (u - shared >= e) i = x + 1, before = e;
    }
    const bool own = u >= shared;
    then_b = own ? first + i : -1;
    then_page = own ? u - shared - before + (p.joined ? a.shared_pages : 0) : u;
    then_id = -1;
    if (k + lane < todo)
      then_id = own ? c.page_table[static_cast<long long>(then_b) * c.max_pages + then_page]
                    : a.shared[then_page];
  };
  look(0);
  look(32);
  int sent = 0;
  auto send = [&] {  // the next page into its slot
    if ((sent & 31) == 0 && sent > 0) look(sent + 32);
    const int id = __shfl_sync(0xffffffffu, now_id, sent & 31), slot = sent % kJobSlots;
    const int tb = __shfl_sync(0xffffffffu, now_b, sent & 31);
    const int page = __shfl_sync(0xffffffffu, now_page, sent & 31);
    const bool ok = id >= 0 && id < c.pages;
    if (lane == 0) {
      sm.task[warp][slot] = make_int2(tb, ok ? page : ~page);
      if (ok) {
        mbar_arrive_expect_tx(&sm.full[warp][slot], kBlk);
        bulk_g2s(sm.ring[warp][slot],
                 c.pool + (static_cast<long long>(id) * c.kv_heads + head) * kBlk, kBlk,
                 &sm.full[warp][slot]);
      } else {
        note_bad(c.err);
        mbar_arrive(&sm.full[warp][slot]);
      }
    }
    ++sent;
  };
  while (sent < todo && sent < kJobSlots) send();
  Piece<D, FMT, DT, 1> k(lane);
  k.start(c, a, p, b, head, tile * kCols);
  const int limits[1][2] = {{k.limit[0][0], k.limit[0][1]}};
  int at = b;  // the sequence whose pages the columns see now
  __syncwarp();
  for (int i = 0; i < todo;) {
    const int s0 = i % kJobSlots, s1 = (i + 1) % kJobSlots;
    const int2 t0 = sm.task[warp][s0];
    const int2 t1 = i + 1 < todo ? sm.task[warp][s1] : make_int2(-2, 0);
    const int page0 = t0.y < 0 ? ~t0.y : t0.y;
    if (t0.x != at) {
      at = t0.x;
      k.only(p, at, limits);
    }
    int there = mbar_sleep(&sm.full[warp][s0], (i / kJobSlots) & 1, &sm.fail) && t0.y >= 0;
    const bool two = t1.x == t0.x;
    if (two) {
      there |= (mbar_sleep(&sm.full[warp][s1], ((i + 1) / kJobSlots) & 1, &sm.fail) && t1.y >= 0) << 1;
      k.template step<2>(sm.ring[warp][s0], sm.ring[warp][s1], page0, there);
    } else {
      k.template step<1>(sm.ring[warp][s0], nullptr, page0, there);
    }
    i += two ? 2 : 1;
    __syncwarp();  // the slots are free
    if (sent < todo) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      send();
      if (two && sent < todo) send();
      __syncwarp();
    }
  }
  settle(&sm.fail);
  // ---- a warp's records, the CTA's, the cluster's ----
  k.close();
  float* mine = reinterpret_cast<float*>(sm.ring[warp]);
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int col = 2 * k.t + x;
    if (k.col0 + col < k.cols) k.put(0, x, mine + col * (D + 4));
  }
  if (lane == 0 && c.err && *static_cast<volatile int*>(&sm.fail)) atomicExch(c.err, sm.fail);
  __syncthreads();
  const int live = min(kCols, k.cols - k.col0);
  auto out = [&](int col, float m, float l, const float* o) {
    const Column cc = column_of(p, b, k.col0 + col);
    put_row<D, DT>(a, p, cc.seq * a.q_tokens + cc.token, head * p.group + cc.head, lane, m, l, o);
  };
  for (int col = warp; col < live; col += kJobWarps) {
    float m = -INFINITY, l = 0.f, o[E] = {};
#pragma unroll
    for (int w = 0; w < kJobWarps; ++w) {
      const float* rec = reinterpret_cast<const float*>(sm.ring[w]) + col * (D + 4);
      float v[E];
      load_lane<E>(rec + lane * E, v);
      join_into<E>(m, l, o, rec[D], rec[D + 1], v);
    }
    if (ctas == 1) {
      out(col, m, l, o);
    } else {
#pragma unroll
      for (int x = 0; x < E; ++x) sm.rec[col][lane * E + x] = o[x];
      if (lane == 0) sm.rec[col][D] = m, sm.rec[col][D + 1] = l;
    }
  }
  if (ctas == 1) return;
  cluster.sync();
  for (int col = rank * kJobWarps + warp; col < live; col += ctas * kJobWarps) {
    float m = -INFINITY, l = 0.f, o[E] = {};
    for (int i = 0; i < ctas; i += 4) {
      float v[4][E], rm[4], rl[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        rl[y] = 0.f;
        if (i + y < ctas) {
          const float* rec = cluster.map_shared_rank(sm.rec[col], i + y);
          load_lane<E>(rec + lane * E, v[y]);
          rm[y] = rec[D], rl[y] = rec[D + 1];
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) join_into<E>(m, l, o, rm[y], rl[y], v[y]);
    }
    out(col, m, l, o);
  }
  cluster.sync();  // the records stay until they have been read
}

}  // namespace

namespace {
Plan attention_plan(const KvqCache& c, int dtype, int q_heads, int q_tokens, int shared_pages) {
  Plan p{};
  p.group = q_heads / c.kv_heads;
  p.rows = q_tokens * p.group;
  p.job_tiles = (p.rows + kCols - 1) / kCols;
  const long long shared_rows = static_cast<long long>(c.seqs) * p.rows;
  const bool more_shared = shared_rows > kCols && (shared_rows + kCols - 1) / kCols * shared_pages >
                               static_cast<long long>(c.seqs) * (c.max_pages - shared_pages);
  const bool pays = c.head_dim == 64 ? p.rows > kCols || more_shared : p.rows > kCols && dtype == kDtBf16;
  p.cols = pays ? 2 * kCols : kCols;
  p.tiles = (p.rows + p.cols - 1) / p.cols;
  p.by_group = Divisor(p.group), p.by_rows = Divisor(p.rows);
  p.by_heads = Divisor(q_heads), p.by_tokens = Divisor(q_tokens);
  p.joined = shared_pages > 0;
  p.group_tiles = static_cast<int>((shared_rows + kCols - 1) / kCols);
  const long long units = c.kv_heads * ((shared_rows + kCols - 1) / kCols) * shared_pages;
  if (dtype == kDtBf16 && shared_rows > kTcRows && units > kTcUnits) {
    p.tc_tiles = static_cast<int>((shared_rows + kRows - 1) / kRows);
    p.tc_jobs = c.kv_heads * p.tc_tiles;
  } else if (shared_pages > 0) {
    p.shared_tiles = static_cast<int>((shared_rows + p.cols - 1) / p.cols);
    p.shared_jobs = c.kv_heads * p.shared_tiles;
    p.shared_units = static_cast<long long>(p.shared_jobs) * (kStart + shared_pages);
  }
  p.jobs = p.shared_jobs + c.seqs * c.kv_heads * p.tiles;
  p.shares = kShares;
  p.bin = c.seqs > kBins ? (c.seqs + kBins - 1) / kBins : 1;
  return p;
}

// CTAs of a job where every job gets a cluster, 0 where the shares are better.
// Lengths are on the device: max_pages bounds them. (16 bf16 heads, 8 kv heads,
// 128 values, int8; us here and by shares.) A single sequence's jobs are all
// alike, so nothing is lost to uneven lengths: up to 11 pages a warp (2,000
// tokens 8.2 and 11.2, 10,000 tokens 15.1 and 15.6, 12,000 tokens 16.9 and 16.4).
// Several sequences: up to 8 (16 of 464 tokens 9.4 and 15.7, 16 of 928 13.4 and
// 19.2, 100 of 128 13.2 and 15.8). With shared pages, where the shares read them
// once for every 8 rows as well and join two parts a row: up to 24 (64 sequences
// of up to 128 tokens behind 1,024, 12 pages a warp, 16.4 and 27.7; 32 behind
// 4,800, 21 pages, 24.8 and 29.5; 128 behind 2,048, 40 pages, 39.0 and 35.8), but 10
// where the clusters leave SMs idle, which the shares do not (8 sequences behind
// 3,200, 8 pages, 13.0 and 13.9; behind 4,800, 11 pages, 15.5 and 14.7).
int job_ctas(const KvqCache& c, const Plan& p, int shared_pages) {
  const long long jobs = p.joined ? static_cast<long long>(c.kv_heads) * p.group_tiles
                                  : static_cast<long long>(c.seqs) * c.kv_heads * p.job_tiles;
  const long long room = 3 * kCtas;  // CTAs that fit at once
  const int seqs = p.joined ? (kCols + p.rows - 1) / p.rows + (kCols % p.rows ? 1 : 0) : 1;  // of a job, at most
  const long long pages = shared_pages + static_cast<long long>(seqs) * (c.max_pages - shared_pages);
  // two pages a warp, or as near as 8 CTAs (16 for a single sequence) come
  int ctas = 1;
  while (ctas < (c.seqs == 1 ? 16 : 8) && ctas * kJobWarps * 2 < pages && jobs * ctas * 2 <= room)
    ctas *= 2;
  const long long each = (pages + ctas * kJobWarps - 1) / (ctas * kJobWarps);  // pages a warp at most
  if (c.seqs == 1 && !p.joined) return jobs * ctas <= room && each <= 11 ? ctas : 0;
  const int most = !p.joined ? 8 : jobs * ctas < kCtas ? 10 : 24;
  return jobs * ctas <= 2 * room && each <= most ? ctas : 0;
}

template <int D, int FMT, int DT, int NT>
cudaError_t launch_attention(const KvqCache& c, const KvqAttention& a, const Plan& p, cudaStream_t s) {
  static std::atomic<unsigned long long> configured{0};
  once_per_device(configured, [&] {
    cudaFuncSetAttribute(kvq_decode_kernel<D, FMT, DT, NT>,
                         cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(DecodeSmem<D>));
  });
  cudaError_t e = cudaSuccess;
  if (p.ctas > 0) {
    constexpr size_t smem = sizeof(JobSmem<D>);
    static std::atomic<unsigned long long> job_configured{0};
    once_per_device(job_configured, [&] {
      cudaFuncSetAttribute(kvq_job_kernel<D, FMT, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           static_cast<int>(smem));
      cudaFuncSetAttribute(kvq_job_kernel<D, FMT, DT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    });
    cudaLaunchConfig_t cfg = {};
    const int jobs = p.joined ? c.kv_heads * p.group_tiles : c.seqs * c.kv_heads * p.job_tiles;
    cfg.gridDim = dim3(static_cast<unsigned>(jobs) * p.ctas);
    cfg.blockDim = dim3(kJobWarps * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.ctas > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kvq_job_kernel<D, FMT, DT>, c, a, p);
  }
  if (p.tc_jobs > 0) {
    e = launch_shared(c, a, p, s);
    if (e != cudaSuccess) return e;
    // starts as the shared pages' CTAs leave, and ends after them
    e = launch_pdl(kvq_decode_kernel<D, FMT, DT, NT>, dim3(kCtas), dim3(kThreads),
                   sizeof(DecodeSmem<D>), s, c, a, p);
  } else {
    kvq_decode_kernel<D, FMT, DT, NT><<<kCtas, kThreads, sizeof(DecodeSmem<D>), s>>>(c, a, p);
    e = cudaGetLastError();
  }
  if (e != cudaSuccess) return e;
  const unsigned rows = static_cast<unsigned>(c.seqs) * a.q_tokens * a.q_heads;
  if (rows >= kManyRows) {
    const int each = static_cast<int>(std::min(32u, (rows + kJoinRows - 1) / kJoinRows));
    const unsigned warps = (rows + each - 1) / each;
    return launch_pdl(each > 1 ? kvq_join_kernel<D, DT, 1, true> : kvq_join_kernel<D, DT, 1>, dim3((warps + kJoinWarps - 1) / kJoinWarps),
                      dim3(kJoinWarps * 32), 0, s, c, a, p, each);
  }
  if (rows <= kFewRows)
    return launch_pdl(kvq_join_kernel<D, DT, 32>, dim3(rows), dim3(1024), 0, s, c, a, p, 1);
  return launch_pdl(kvq_join_kernel<D, DT, kJoinWarps>, dim3(rows), dim3(kJoinWarps * 32), 0, s, c, a, p,
                    1);
}
}  // namespace

size_t kvq_attention_workspace(const KvqCache& c, int q_heads, int q_tokens, int shared_pages) {
  // enough for either type of rows
  size_t most = 0;
  for (int dtype : {kDtF32, kDtBf16}) {
    const Plan p = attention_plan(c, dtype, q_heads, q_tokens, shared_pages);
    const size_t n = p.directory_bytes() + (p.record_floats(c.head_dim) + p.tc_record_floats(c.head_dim)) *
                                               sizeof(float);
    most = n > most ? n : most;
  }
  return most;
}

cudaError_t op_kvq_attention(const KvqCache& c, const KvqAttention& a, cudaStream_t s) {
  Plan p = attention_plan(c, a.dtype, a.q_heads, a.q_tokens, a.shared_pages);
  p.ctas = job_ctas(c, p, a.shared_pages);
  p.q_vec = rows_aligned(a.q, a.q, a.dtype, a.q_stride, a.q_stride);
  p.out_vec = rows_aligned(a.out, a.out, a.dtype, a.out_stride, a.out_stride);
  cudaError_t e = cudaSuccess;
  kvq_dispatch(a.dtype, c.format, c.head_dim, true, [&](auto dt, auto fmt, auto d, auto vec) {
    if constexpr (vec) {
      if (p.cols > kCols)
        e = launch_attention<d, fmt, dt, dt == kDtBf16 || d == 64 ? 2 : 1>(c, a, p, s);
      else
        e = launch_attention<d, fmt, dt, 1>(c, a, p, s);
    }
  });
  return e;
}

}  // namespace orx
