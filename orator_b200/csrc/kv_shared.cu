// Attention of a whole batch over the pages that all its sequences share, on
// tcgen05: per kv head, the query rows of every sequence are the 128 rows of
// one tile, so each shared page is read once per 128 rows, and
//   S = Q K^T  (128 rows x 64 keys, depth D),   O += P V  (depth 64)
// are full-size tensor-core products. Bound by the products and, as much, by
// one exponential per score (16 a clock and SM).
//
// Reference, scales and fp16 operands are the decode kernel's (kv_attention.cu):
// codes are exact in fp16, K's scale multiplies the score, V's the
// probability, a row's reference r follows the largest z_j + log2 vs_j and
// rises only when it is passed by 2^4, so that p_j vs_j keeps fp16's digits down
// to 2^-24 of the row's largest and counts down to 2^-35 of it.
//
// One CTA per SM takes an equal share of all (head, 128 rows, 64 keys) tiles in
// a row; the part of a (head, 128 rows) job that it has is a segment.
//   warps 0-15   softmax: two teams of eight warps on the even and the odd
//                tiles of a segment, each with an O and references of its own,
//                two threads a row, 32 keys each; one team's exponentials run
//                while the other waits for products or takes maxima
//   warps 16-23  turn codes into fp16 tiles, 128-byte swizzle, K as [key][D] for
//                S (D contiguous: K-major) and V as [key][D] for O (MN-major)
//   warp 24      fetches raw blocks, 4 pages a tile, by bulk copies
//   warp 25      issues the products, S two tiles ahead of O;
//                Q and P are operands in TMEM, which leaves shared memory's
//                bandwidth to K and V
// TMEM columns: Q 64 | S 2 x 64 | P 2 x 32 | O 2 x 128 = 512.
#include <algorithm>

#include "kv_quant.cuh"

namespace orx {
using namespace kvq;
namespace {

constexpr int kSoftWarps = 16, kConvWarps = 8;
constexpr int kParts = 2, kKeys = kTile / kParts;  // threads of a row in a team, keys of each
constexpr int kSlices = kSoftWarps / 4;             // threads of a row in both: of Q and O they take D / 4
constexpr int kFetchWarp = kSoftWarps + kConvWarps, kMmaWarp = kFetchWarp + 1;
constexpr int kThreads = (kFetchWarp + 4) * 32;  // warpgroups are whole
// Registers a thread: 72 at launch (65,536 / 896, in eights), then moved to the softmax:
// 512 x 88 + 256 x 56 + 128 x 40 = 64,512 = 896 x 72.
constexpr int kSoftRegs = 88, kConvRegs = 56, kRestRegs = 40;
constexpr int kRaw = 3, kKv = 4;  // stages of raw blocks and of fp16 tiles
constexpr int kPages = kTile / kPage;
// Two warps rescale their O when one of their 32 rows rises. 256 sessions behind 16,384 tokens, the
// whole call: 122 us with room for 2^4, and 121, 119, 117 and 115 with 2^6, 2^8, 2^10 and 2^12, each
// of which takes as much off the lower end of p vs; what is lost there is lost once a key.
constexpr int kColQ = 0, kColS = 64, kColP = 192, kColO = 256;  // S, P, O: one after the other for the teams

template <int D>
struct SharedSmem {
  alignas(1024) uint8_t k[kKv][kTile * D * 2];  // halves of 64 values: [64 keys][128 bytes]
  alignas(1024) uint8_t v[kKv][kTile * D * 2];
  alignas(128) uint8_t raw[kRaw][kPages * kvq_block_bytes(D)];
  alignas(16) float ks[kKv][kTile], vs[kKv][kTile], ve[kKv][kTile];
  int fine[kRaw], kv_fine[kKv];  // bit i: page i is there
  float part[kSlices][kRows], ref[2][kRows];  // what the threads of a row tell one another
  uint64_t raw_full[kRaw], raw_empty[kRaw], kv_full[kKv], kv_empty[kKv];
  uint64_t s_full[2], s_free[2], p_full[2], o_done[2], q_full;
  uint32_t tmem;
  int fail;
};

__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  uint64_t d = (addr >> 4) & 0x3FFF;
  d |= static_cast<uint64_t>((lead >> 4) & 0x3FFF) << 16;
  d |= static_cast<uint64_t>((stride >> 4) & 0x3FFF) << 32;
  d |= static_cast<uint64_t>(1) << 46;  // descriptor version (sm_100)
  d |= static_cast<uint64_t>(2) << 61;  // 128-byte swizzle
  return d;
}
// D[128 x N] (+)= A[128 x 16] B[N x 16]^T, A in TMEM.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// 16 columns of this warp's 32 lanes, complete on return.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      " tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void soft_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(kSoftWarps * 32) : "memory");
}
// The two warps of a team that hold the same rows.
__device__ __forceinline__ void pair_barrier(int id) {
  asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory");
}
__device__ __forceinline__ bool pair_barrier_or(int id, bool v) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, %2, 64, p;\n"
      " selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "r"(id)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The tiles of this CTA's share in order, cut at the ends of jobs.
struct Segments {
  int tiles;  // key tiles of a job
  long long at, end;
  int job, t0, n;
  __device__ __forceinline__ bool next() {
    if (at >= end) return false;
    job = static_cast<int>(at / tiles);
    t0 = static_cast<int>(at - static_cast<long long>(job) * tiles);
    n = static_cast<int>(min(static_cast<long long>(tiles - t0), end - at));
    at += n;
    return true;
  }
};

template <int D, int FMT>
__global__ void __launch_bounds__(kThreads, 1) kvq_shared_kernel(KvqCache c, KvqAttention a, Plan p) {
  constexpr int kBlk = kvq_block_bytes(D);
  constexpr int kHalves = D / 64, kHalfBytes = kTile * 128;
  extern __shared__ uint8_t shared_raw[];
  SharedSmem<D>& sm = *reinterpret_cast<SharedSmem<D>*>(
      (reinterpret_cast<uintptr_t>(shared_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == kMmaWarp) {
    if (lane == 0) {
      sm.fail = 0;
      for (int i = 0; i < kRaw; ++i) mbar_init(&sm.raw_full[i], 1), mbar_init(&sm.raw_empty[i], kConvWarps);
      for (int i = 0; i < kKv; ++i) mbar_init(&sm.kv_full[i], kConvWarps), mbar_init(&sm.kv_empty[i], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&sm.s_full[i], 1);
        mbar_init(&sm.s_free[i], kSoftWarps / 2);
        mbar_init(&sm.p_full[i], kSoftWarps / 2);
        mbar_init(&sm.o_done[i], 1);
      }
      mbar_init(&sm.q_full, kSoftWarps);
      fence_mbar_init();
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&sm.tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  pdl_trigger();
  const uint32_t tmem = sm.tmem;
  int* fail = &sm.fail;
  const int tiles = (a.shared_pages + kPages - 1) / kPages;
  const Share share = share_of(blockIdx.x, static_cast<long long>(p.tc_jobs) * tiles, kCtas);
  Segments seg{tiles, share.start, share.start + share.count, 0, 0, 0};

  if (warp >= kFetchWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRestRegs));
  if (warp == kFetchWarp) {
    // ---- raw blocks, 4 pages a tile; page ids 32 at a time, one batch ahead ----
    int i = 0;
    while (seg.next()) {
      const int head = seg.job / p.tc_tiles, page0 = seg.t0 * kPages;
      const int pages = min(seg.n * kPages, a.shared_pages - page0);
      auto ids = [&](int k) { return k + lane < pages ? a.shared[page0 + k + lane] : -1; };
      int now = ids(0), then = ids(32);
      for (int t = 0; t < seg.n; ++t, ++i) {
        const int at = t * kPages % 32;
        if (t > 0 && at == 0) {
          now = then;
          then = ids(t * kPages + 32);
        }
        const int s = i % kRaw;
        const bool ok = i < kRaw || mbar_sleep(&sm.raw_empty[s], (i / kRaw - 1) & 1, fail);
        const int id = __shfl_sync(0xffffffffu, now, (at + lane) & 31);
        const bool asked = lane < kPages && t * kPages + lane < pages;
        const bool fine = ok && asked && id >= 0 && id < c.pages;
        if (asked && !(id >= 0 && id < c.pages)) note_bad(c.err);
        const unsigned mask = __ballot_sync(0xffffffffu, fine);
        if (lane == 0) {
          sm.fine[s] = static_cast<int>(mask);
          if (mask)
            mbar_arrive_expect_tx(&sm.raw_full[s], __popc(mask) * kBlk);
          else
            mbar_arrive(&sm.raw_full[s]);
        }
        __syncwarp();
        if (fine)
          bulk_g2s(sm.raw[s] + lane * kBlk,
                   c.pool + (static_cast<long long>(id) * c.kv_heads + head) * kBlk, kBlk,
                   &sm.raw_full[s]);
      }
    }
  } else if (warp == kMmaWarp) {
    // ---- products: S of tile i goes out before O of tile i - 1 ----
    // All lanes run the loop, one issues: what is the same in all of them stays in uniform
    // registers (an MMA costs 100 cycles to issue where a single lane runs the loop).
    constexpr uint32_t kIdS = (1u << 4) | (static_cast<uint32_t>(kTile / 8) << 17) | (8u << 24);
    constexpr uint32_t kIdO =
        (1u << 4) | (1u << 16) | (static_cast<uint32_t>(D / 8) << 17) | (8u << 24);
    constexpr uint32_t kStage = kTile * D * 2;
    const bool leader = elect_one();
    const uint64_t kd = smem_desc(smem_u32(sm.k[0]), 16, 1024);
    const uint64_t vd = smem_desc(smem_u32(sm.v[0]), kHalfBytes, 1024);
    int i = 0, segs = 0;
    uint32_t begun = 0, s_phase = 0, p_phase = 0;  // a bit for each team
    while (seg.next()) {
      mbar_sleep(&sm.q_full, segs++ & 1, fail);
      fence_after();
      auto issue_s = [&](int t) {
        const int s = (i + t) % kKv, w = t & 1;
        mbar_sleep(&sm.kv_full[s], ((i + t) / kKv) & 1, fail);
        // the team has the scores of its last tile in registers
        if (begun >> w & 1) {
          mbar_sleep(&sm.s_free[w], s_phase >> w & 1, fail);
          s_phase ^= 1u << w;
        }
        begun |= 1u << w;
        fence_after();
        const uint64_t desc = kd + (s * kStage >> 4);
        if (leader) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ts(tmem + kColS + w * kTile, tmem + kColQ + 8 * k,
                   desc + ((k / 4 * kHalfBytes + k % 4 * 32) >> 4), kIdS, k > 0);
          commit(&sm.s_full[w]);
        }
        __syncwarp();
      };
      issue_s(0);
      if (seg.n > 1) issue_s(1);
      for (int t = 0; t < seg.n; ++t) {
        // a team's next scores before its last product, so that it finds them ready
        if (t + 2 < seg.n) issue_s(t + 2);
        const int s = (i + t) % kKv, w = t & 1;
        mbar_sleep(&sm.p_full[w], p_phase >> w & 1, fail);
        p_phase ^= 1u << w;
        fence_after();
        const uint64_t desc = vd + (s * kStage >> 4);
        const bool more = t > 1;
        if (leader) {
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k)
            mma_ts(tmem + kColO + w * D, tmem + kColP + w * (kTile / 2) + 8 * k,
                   desc + (k * 16 * 128 >> 4), kIdO, more || k > 0);
          commit(&sm.o_done[w]);
          commit(&sm.kv_empty[s]);
        }
        __syncwarp();
      }
      i += seg.n;
    }
  }
  } else if (warp >= kSoftWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kConvRegs));
    // ---- codes to fp16 tiles ----
    const int ct = threadIdx.x - kSoftWarps * 32;
    int i = 0;
    while (seg.next()) {
      for (int t = 0; t < seg.n; ++t, ++i) {
        const int rs = i % kRaw, s = i % kKv;
        mbar_sleep(&sm.raw_full[rs], (i / kRaw) & 1, fail);
        if (i >= kKv) mbar_sleep(&sm.kv_empty[s], (i / kKv - 1) & 1, fail);
        const uint8_t* raw = sm.raw[rs];
        if (ct < kTile) {
          const float* sc =
              reinterpret_cast<const float*>(raw + ct / kPage * kBlk + 2 * kPage * D) + ct % kPage;
          const int fine = sm.fine[rs];
          const bool there = fine >> (ct / kPage) & 1;
          const float vs = there ? sc[kPage] : 0.f;
          sm.ks[s][ct] = there ? sc[0] : 0.f;
          sm.vs[s][ct] = vs;
          sm.ve[s][ct] = scale_exponent(vs);
          if (ct == 0) sm.kv_fine[s] = fine;
        }
        // 16 codes at a time, a row by neighbouring lanes, kAtOnce rows at once
        constexpr int kChunks = D / 16, kAtOnce = kConvWarps * 32 / kChunks;
        const int ch = ct % kChunks, key0 = ct / kChunks;
        // the lanes of the second half of a row store their second 8 values first, as both halves'
        // first ones lie at the same banks
        const bool swap = ch / 4 & 1;
        const uint8_t* src0 = raw + key0 / kPage * kBlk + key0 % kPage * D + ch * 16;
        const int at0 = ch / 4 * kHalfBytes + key0 * 128 + ((ch % 4 * 2 + (swap ? 1 : 0)) ^ (key0 & 7)) * 16;
        const int other = at0 & 16 ? -16 : 16;  // to the 16 bytes beside, swizzled
#pragma unroll
        for (int kind = 0; kind < 2; ++kind) {
          uint8_t* dst0 = (kind ? sm.v[s] : sm.k[s]) + at0;
#pragma unroll
          for (int y = 0; y < kTile; y += kAtOnce) {
            const uint4 q = *reinterpret_cast<const uint4*>(src0 + y / kPage * kBlk + kind * kPage * D);
            uint32_t h[8];
            codes_to_half<FMT>(swap ? q.z : q.x, h[0], h[1]);
            codes_to_half<FMT>(swap ? q.w : q.y, h[2], h[3]);
            codes_to_half<FMT>(swap ? q.x : q.z, h[4], h[5]);
            codes_to_half<FMT>(swap ? q.y : q.w, h[6], h[7]);
            if (FMT == kKvqE4m3 && kind) {
              // a slot that was never written may hold a NaN's code, which 0 * would keep (and is a key
              // seen, so that a NaN's code that something else put into the pool counts as 448)
              const __half2 top = __half2half2(__ushort_as_half(0x5F00));  // 448
#pragma unroll
              for (int z = 0; z < 8; ++z) {
                const __half2 m = __hmin2(*reinterpret_cast<__half2*>(&h[z]), top);
                h[z] = *reinterpret_cast<const uint32_t*>(&m);
              }
            }
            *reinterpret_cast<uint4*>(dst0 + y * 128) = make_uint4(h[0], h[1], h[2], h[3]);
            *reinterpret_cast<uint4*>(dst0 + y * 128 + other) = make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&sm.kv_full[s]);
          mbar_arrive(&sm.raw_empty[rs]);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
    // ---- softmax: row `row`, keys [kKeys part, kKeys (part + 1)) of the team's tiles ----
    const int slice = warp >> 2, team = slice & 1, part = slice >> 1, row = (warp & 3) * 32 + lane;
    const int pair = 2 + (warp & 3) * 2 + team;  // the named barrier of its two warps
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) * 32 << 16);
    constexpr int kCols = D / kSlices;  // of Q and O, this thread's
    uint32_t done = 0;  // tiles of this team
    int i = 0;
    while (seg.next()) {
      const int head = seg.job / p.tc_tiles;
      const int col = (seg.job - head * p.tc_tiles) * kRows + row;
      const bool live = col < c.seqs * p.rows;
      const Column cc = column_of(p, -1, live ? col : 0);
      // the row's queries: scaled to fp16's upper end, into TMEM
      const long long at = (static_cast<long long>(cc.seq) * a.q_tokens + cc.token) * a.q_stride +
                           static_cast<long long>(head * p.group + cc.head) * D + slice * kCols;
      uint32_t q[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 8; ++j) {
        const uint4 w = p.q_vec ? load_raw<kDtBf16, true>(a.q, at + 8 * j) : load_raw<kDtBf16, false>(a.q, at + 8 * j);
        q[4 * j] = w.x, q[4 * j + 1] = w.y, q[4 * j + 2] = w.z, q[4 * j + 3] = w.w;
      }
      const int limit =
          live ? min(seq_len(c, a, cc.seq) - a.q_tokens + cc.token + 1, a.shared_pages * kPage)
               : a.shared_pages * kPage;
      const int all_see = __reduce_min_sync(0xffffffffu, limit);
      uint32_t most = 0;
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j)
        asm("max.NaN.bf16x2 %0, %0, %1;" : "+r"(most) : "r"(q[j] & 0x7fff7fffu));
      sm.part[slice][row] = __uint_as_float(max(most << 16, most & 0xffff0000u));
      soft_barrier();
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < kSlices; ++j) amax = max(amax, __float_as_uint(sm.part[j][row]));
      if (!live) amax = 0;
      const int up = amax ? 14 - (static_cast<int>(amax >> 23) - 127) : 0;
      const float f1 = amax >= 0x7f800000u ? NAN : __uint_as_float((127 + up / 2) << 23);
      const float f2 = __uint_as_float((127 + up - up / 2) << 23);
      const float qf = a.scale * 1.4426950408889634f * __uint_as_float((127 - up / 2) << 23) *
                       __uint_as_float((127 - (up - up / 2)) << 23);
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j)
        q[j] = live ? pack_half(bf_lo(q[j]) * f1 * f2, bf_hi(q[j]) * f1 * f2) : 0u;
#pragma unroll
      for (int j = 0; j < kCols / 2; j += 8) tmem_st8(lanes + kColQ + slice * kCols / 2 + j, q + j);
      st_wait();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sm.q_full);
      soft_barrier();  // sm.part has been read

      float r = -INFINITY, l = 0.f;
      for (int t = team; t < seg.n; t += 2) {
        const int s = (i + t) % kKv;
        mbar_sleep(&sm.kv_full[s], ((i + t) / kKv) & 1, fail);  // the scales
        const float4* ks = reinterpret_cast<const float4*>(&sm.ks[s][part * kKeys]);
        const float4* vs = reinterpret_cast<const float4*>(&sm.vs[s][part * kKeys]);
        const int pos = (seg.t0 + t) * kTile + part * kKeys, fine = sm.kv_fine[s];
        const float4* ve = reinterpret_cast<const float4*>(&sm.ve[s][part * kKeys]);
        const int there = fine >> (part * kKeys / kPage) & 3;  // of its two pages
        // some row of the warp does not see some key
        const bool edge = pos + kKeys > all_see || there != 3;
        const float rk = r == -INFINITY ? 0.f : r - kLift;
        mbar_sleep(&sm.s_full[team], done & 1, fail);
        fence_after();
        uint32_t x[kKeys];
        tmem_ld32(lanes + kColS + team * kTile + part * kKeys, x);
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.s_free[team]);
        float2 z[kKeys / 2];
        const float2 q2 = make_float2(qf, qf), r2 = make_float2(-rk, -rk);
#pragma unroll
        for (int j = 0; j < kKeys / 4; ++j) {
          const float4 k4 = ks[j];
          z[2 * j] = fma2(mul2(make_float2(__uint_as_float(x[4 * j]), __uint_as_float(x[4 * j + 1])),
                               make_float2(k4.x, k4.y)), q2, r2);
          z[2 * j + 1] = fma2(mul2(make_float2(__uint_as_float(x[4 * j + 2]), __uint_as_float(x[4 * j + 3])),
                                   make_float2(k4.z, k4.w)), q2, r2);
        }
        if (edge) {
          const int seen = limit - pos;
#pragma unroll
          for (int j = 0; j < kKeys / 2; ++j) {
            const bool page = there >> (2 * j / kPage) & 1;
            if (2 * j >= seen || !page) z[j].x = -INFINITY;
            if (2 * j + 1 >= seen || !page) z[j].y = -INFINITY;
          }
        }
        float t4[4];
#pragma unroll
        for (int j = 0; j < kKeys / 4; ++j) {
          const float4 e4 = ve[j];
          const float2 a = add2(z[2 * j], make_float2(e4.x, e4.y)), b = add2(z[2 * j + 1], make_float2(e4.z, e4.w));
          const int x = 2 * (j & 1);
          t4[x] = j < 2 ? fmaxf(a.x, a.y) : max3(t4[x], a.x, a.y);
          t4[x + 1] = j < 2 ? fmaxf(b.x, b.y) : max3(t4[x + 1], b.x, b.y);
        }
        float top = fmaxf(max3(t4[0], t4[1], t4[2]), t4[3]);
        top += rk;  // of z + log2 vs
        if (pair_barrier_or(pair, top > r + kSlack)) {
          // ---- some row's reference rises: the rows' maxima, and O where it does ----
          sm.part[slice][row] = top;
          pair_barrier(pair);
          top = fmaxf(top, sm.part[slice ^ 2][row]);
          const bool rise = top > r + kSlack;
          const float h = rise ? ex2_half(r - top) : 1.0f, f = h * h;  // 0 for the first
          const float shift = rise ? rk - (top - kLift) : 0.f;
#pragma unroll
          for (int j = 0; j < kKeys / 2; ++j) z[j] = add2(z[j], make_float2(shift, shift));
          if (rise) {
            r = top;
            l = l * h * h;
          }
          if (t > 1) {
            mbar_sleep(&sm.o_done[team], (done - 1) & 1, fail);
            fence_after();
            // the two warps take half of the columns each
#pragma unroll 1
            for (int d = part * (D / 2); d < (part + 1) * (D / 2); d += 16) {
              uint32_t o[16];
              tmem_ld16(lanes + kColO + team * D + d, o);
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st16(lanes + kColO + team * D + d, o);
            }
          }
          pair_barrier(pair);  // the maxima have been read
        }
        uint32_t pk[kKeys / 2];
        float2 sum = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < kKeys / 4; ++j) {
          const float4 v4 = vs[j];
          const float2 e0 = make_float2(ex2(z[2 * j].x), ex2(z[2 * j].y));
          const float2 e1 = make_float2(ex2(z[2 * j + 1].x), ex2(z[2 * j + 1].y));
          sum = add2(sum, add2(e0, e1));
          float2 p0 = mul2(e0, make_float2(v4.x, v4.y)), p1 = mul2(e1, make_float2(v4.z, v4.w));
          if (edge) {  // a V scale may be NaN
            if (z[2 * j].x == -INFINITY) p0.x = 0.f;
            if (z[2 * j].y == -INFINITY) p0.y = 0.f;
            if (z[2 * j + 1].x == -INFINITY) p1.x = 0.f;
            if (z[2 * j + 1].y == -INFINITY) p1.y = 0.f;
          }
          pk[2 * j] = pack_half(p0.x, p0.y);
          pk[2 * j + 1] = pack_half(p1.x, p1.y);
        }
        l += sum.x + sum.y;
        if (t > 1) {
          mbar_sleep(&sm.o_done[team], (done - 1) & 1, fail);  // P's place has been read
          fence_after();
        }
        tmem_st16(lanes + kColP + team * (kTile / 2) + part * (kKeys / 2), pk);
        st_wait();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.p_full[team]);
        ++done;
      }
      // ---- the segment's record: both teams' O, a quarter of the columns a thread ----
      i += seg.n;
      if (team < seg.n) mbar_sleep(&sm.o_done[team], (done - 1) & 1, fail);
      sm.part[slice][row] = l;
      if (part == 0) sm.ref[team][row] = r;
      fence_before();
      soft_barrier();
      fence_after();
      const float r0 = sm.ref[0][row], r1 = sm.ref[1][row], top = fmaxf(r0, r1);
      const float l0 = sm.part[0][row] + sm.part[2][row], l1 = sm.part[1][row] + sm.part[3][row];
      const float h0 = l0 == 0.f ? 0.f : ex2_half(r0 - top), h1 = l1 == 0.f ? 0.f : ex2_half(r1 - top);
      const float w0 = h0 * h0, w1 = h1 * h1;
      float* rec = p.tc_records(a.ws, D) +
                   static_cast<long long>(blockIdx.x + seg.job) * kRows * (D + 4);
#pragma unroll 1
      for (int d = slice * kCols; d < (slice + 1) * kCols; d += 16) {
        uint32_t o0[16], o1[16];
        tmem_ld16(lanes + kColO + d, o0);
        tmem_ld16(lanes + kColO + D + d, o1);
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          v[j] = (l0 == 0.f ? 0.f : __uint_as_float(o0[j]) * w0) +
                 (l1 == 0.f ? 0.f : __uint_as_float(o1[j]) * w1);
#pragma unroll
        for (int j = 0; j < 16; j += 4)
          *reinterpret_cast<float4*>(rec + (d + j) / 8 * (kRows * 8) + row * 8 + j % 8) =
              make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
      }
      if (slice == 0) {
        // l and O are both 2^kLift too large
        const float sum = (l0 == 0.f ? 0.f : l0 * h0 * h0) + (l1 == 0.f ? 0.f : l1 * h1 * h1);
        *reinterpret_cast<float2*>(rec + kRows * D + 2 * row) = make_float2(top - kLift, sum);
        if (row == 0) {
          int* dir = p.directory(a.ws) + 2 * (p.jobs + seg.job);
          if (seg.t0 == 0) dir[0] = blockIdx.x;
          if (seg.t0 + seg.n == tiles) dir[1] = blockIdx.x;
        }
      }
      fence_before();
      soft_barrier();  // O and the rows' numbers may be written again
      fence_after();
    }
  }
  settle(fail);
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  if (threadIdx.x == 0 && sm.fail && c.err) atomicExch(c.err, sm.fail);
}

template <int D, int FMT>
cudaError_t launch(const KvqCache& c, const KvqAttention& a, const Plan& p, cudaStream_t s) {
  constexpr size_t smem = sizeof(SharedSmem<D>) + 1024;
  static_assert(smem <= 227 * 1024, "shared memory");
  static std::atomic<unsigned long long> configured{0};
  once_per_device(configured, [&] {
    cudaFuncSetAttribute(kvq_shared_kernel<D, FMT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                         static_cast<int>(smem));
  });
  kvq_shared_kernel<D, FMT><<<kCtas, kThreads, smem, s>>>(c, a, p);
  return cudaGetLastError();
}

}  // namespace

namespace kvq {
cudaError_t launch_shared(const KvqCache& c, const KvqAttention& a, const Plan& p, cudaStream_t s) {
  if (c.head_dim == 64)
    return c.format == kKvqInt8 ? launch<64, kKvqInt8>(c, a, p, s) : launch<64, kKvqE4m3>(c, a, p, s);
  return c.format == kKvqInt8 ? launch<128, kKvqInt8>(c, a, p, s) : launch<128, kKvqE4m3>(c, a, p, s);
}
}  // namespace kvq

}  // namespace orx
