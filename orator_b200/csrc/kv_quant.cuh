// What the kernels of the 8-bit paged KV cache share: block layout helpers,
// code conversions, the attention's plan of work and its columns.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace orx {
namespace kvq {

// A bad index, which is skipped, does not hide a wait that ran out, after which outputs are missing.
__device__ __forceinline__ void note_bad(int* err) {
  if (err) atomicCAS(err, kErrNone, kErrBadIndex);
}

__device__ __forceinline__ float load_f(const void* p, int dtype, long long i) {
  return dtype == kDtBf16 ? bf2f(static_cast<const uint16_t*>(p)[i])
                          : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_f(void* p, int dtype, long long i, float v) {
  if (dtype == kDtBf16)
    static_cast<uint16_t*>(p)[i] = f2bf(v);
  else
    static_cast<float*>(p)[i] = v;
}

template <int DT>
struct Wide {
  static constexpr int kVals = DT == kDtBf16 ? 8 : 4;
};

// kVals values as they lie in memory, in one load where they are aligned.
template <int DT, bool VEC>
__device__ __forceinline__ uint4 load_raw(const void* p, long long i) {
  if (DT == kDtBf16) {
    const uint16_t* q = static_cast<const uint16_t*>(p) + i;
    if (VEC) return __ldg(reinterpret_cast<const uint4*>(q));
    return make_uint4(q[0] | q[1] << 16, q[2] | q[3] << 16, q[4] | q[5] << 16, q[6] | q[7] << 16);
  }
  const uint32_t* q = static_cast<const uint32_t*>(p) + i;
  if (VEC) return __ldg(reinterpret_cast<const uint4*>(q));
  return make_uint4(q[0], q[1], q[2], q[3]);
}
template <int DT>
__device__ __forceinline__ void unpack_raw(const uint4& w, float* x) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (DT == kDtBf16)
      x[2 * j] = bf_lo(r[j]), x[2 * j + 1] = bf_hi(r[j]);
    else
      x[j] = __uint_as_float(r[j]);
  }
}
template <int DT, bool VEC>
__device__ __forceinline__ void load_vals(const void* p, long long i, float* x) {
  unpack_raw<DT>(load_raw<DT, VEC>(p, i), x);
}

constexpr float kSlack = 4.0f;
constexpr float kLift = 10.0f;        // p is held 2^10 too large: p vs at most 2^15, down to 2^-35 of it
// log2 of V scales counts from here, or r would leave p no range: p is at most 2^94, and 2^33 of them
// add up. Products of rows whose scales are all smaller keep fp16's digits down to scales of 2^-104,
// and count down to 2^-115.
constexpr float kLeastV = -80.0f;
constexpr float kLog2e = 1.4426950408889634f;

// What a V scale counts as in a row's reference: floor of its log2 (2^23 + exponent as a float, less
// 2^23 + 127), kLeastV at least. One that is no number poisons the products, but must not raise the
// reference, or the sum of probabilities would lose the other keys.
__device__ __forceinline__ float scale_exponent(float vs) {
  const float e = __uint_as_float(0x4B000000u | (__float_as_uint(vs) >> 23)) - 8388735.0f;
  return e > 127.0f ? kLeastV : fmaxf(e, kLeastV);
}

// Bounded wait that sleeps in the barrier unit (about 4 us a try, whatever time is asked for), so
// that waiting warps take no issue slots from working ones. False after kWaitLimitNs, or at once when
// another wait already failed.
__device__ __forceinline__ bool mbar_sleep_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(1000000)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ uint32_t global_ns_low() {  // 4 s in all
  uint32_t t;
  asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(t));
  return t;
}
__device__ __forceinline__ bool mbar_sleep(uint64_t* bar, uint32_t parity, int* fail) {
  if (mbar_sleep_try(bar, parity)) return true;
  const uint32_t t0 = global_ns_low();
  while (!mbar_sleep_try(bar, parity)) {
    if (*reinterpret_cast<volatile int*>(fail) != 0) return false;
    if (global_ns_low() - t0 > kWaitLimitNs) {
      atomicExch(fail, kErrWaitTimeout);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// After a wait that ran out: time for copies and products under way to land
// before the CTA gives its memory back.
__device__ __forceinline__ void settle(const int* fail) {
  if (*reinterpret_cast<const volatile int*>(fail) == 0) return;
  for (const unsigned long long t0 = global_ns(); global_ns() - t0 < 10000000;) __nanosleep(100000);
}

constexpr int kCtas = 148;            // one per SM
constexpr int kRows = 128;            // query rows of a tile of the shared pages on tcgen05
constexpr int kTile = 64;             // and its keys

// Quotients n / d, 0 <= n < 2^31, by a multiplication (T. Granlund and P. L.
// Montgomery, "Division by invariant integers using multiplication", 1994).
struct Divisor {
  uint32_t d, mul;
  int shift;
  Divisor() = default;
  explicit Divisor(int by) : d(by), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = static_cast<uint32_t>((((1ull << shift) - d) << 32) / d + 1);
  }
  __device__ __forceinline__ int of(int n) const {
    return static_cast<int>((__umulhi(mul, n) + static_cast<uint32_t>(n)) >> shift);
  }
};

struct Plan {
  Divisor by_group, by_rows, by_heads, by_tokens;  // group, rows; the call's query heads and tokens
  int group, rows;        // query heads per kv head; query rows of one sequence and kv head
  int cols;               // of a job in the decode kernel: 8 or 16 query rows
  int tiles, shared_tiles, job_tiles;  // of `cols` rows; of 8, for the clusters
  int shared_jobs;        // of the shared pages in the decode kernel: (head, `cols` rows)
  long long shared_units;
  int bin;                // sequences per run
  bool q_vec, out_vec;    // rows start on 16 bytes
  bool joined;            // every row has pieces of the shared pages and of its own
  int tc_tiles, tc_jobs;  // of the shared pages on tcgen05: row tiles a head, (head, row tile)
  int shares;             // of the decode kernel: one per consumer warp
  int ctas;               // > 0: every job gets a cluster of that many, and nothing else runs
  int group_tiles;        // then, with shared pages: tiles of 8 rows of all sequences a head
  // The workspace: first and last share of every job -- the decode kernel's,
  // then tcgen05's --, the decode pieces' records (`cols` rows at share + job), and
  // tcgen05's (128 rows at CTA + job). A row's record: D values, r, l, padding;
  // in tcgen05's the values lie [D / 8][128 rows][8] and behind them (r, l) of
  // the rows, so that threads that hold a row each write, and a warp that reads
  // one row reads, whole sectors.
  int jobs;
  __host__ __device__ size_t directory_bytes() const {
    return (static_cast<size_t>(jobs + tc_jobs) * 8 + 15) / 16 * 16;
  }
  __host__ __device__ size_t record_floats(int D) const {
    return static_cast<size_t>(shares + jobs) * cols * (D + 4);
  }
  __host__ __device__ size_t tc_record_floats(int D) const {
    return tc_jobs > 0 ? static_cast<size_t>(kCtas + tc_jobs) * kRows * (D + 4) : 0;
  }
  __device__ int* directory(void* ws) const { return static_cast<int*>(ws); }
  __device__ float* records(void* ws) const {
    return reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + directory_bytes());
  }
  __device__ float* tc_records(void* ws, int D) const { return records(ws) + record_floats(D); }
};

__device__ __forceinline__ int own_pages(const KvqCache& c, const KvqAttention& a, int b) {
  int n = a.lens[b];
  n = n < 0 ? 0 : n;
  const long long cap = static_cast<long long>(c.max_pages) * kPage;
  if (n > cap) n = static_cast<int>(cap);
  n = (n + kPage - 1) / kPage - a.shared_pages;
  return n > 0 ? n : 0;
}
__device__ __forceinline__ int seq_len(const KvqCache& c, const KvqAttention& a, int b) {
  const int n = a.lens[b];
  const long long cap = static_cast<long long>(c.max_pages) * kPage;
  if (n < 0 || n > cap) {
    note_bad(c.err);
    return n < 0 ? 0 : static_cast<int>(cap);
  }
  return n;
}

// `units` cut into n shares, the first units % n of which have one more than
// the others: [start, start + count) of share w.
struct Share {
  long long start;
  int count;
};
__device__ __forceinline__ Share share_of(int w, long long units, int n) {
  if (units <= n) return {w, w < units ? 1 : 0};
  const long long each = units / n;
  const int more = static_cast<int>(units - each * n);
  return {w * each + min(w, more), static_cast<int>(each) + (w < more ? 1 : 0)};
}

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^(d / 2), d <= 0: sums of probabilities are scaled by 2^d in two steps, as they may be large and 2^d
// too small for a number where the V scales are far apart.
__device__ __forceinline__ float ex2_half(float d) { return ex2(0.5f * d); }
// ln(l 2^r): the exponent of l goes to r first, as the two may be far apart.
__device__ __forceinline__ float ln_sum(float r, float l) {
  if (!(l < INFINITY)) return l + r;
  const float e = static_cast<float>(static_cast<int>(__float_as_uint(l) >> 23) - 127);
  const float f = __uint_as_float((__float_as_uint(l) & 0x7fffffu) | 0x3f800000u);
  return ((r + e) + log2f(f)) * 0.6931471805599453f;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_half(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// Bytes 0, 1 and 2, 3 of w as pairs of fp16.
template <int FMT>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& h01, uint32_t& h23) {
  if (FMT == kKvqInt8) {  // 0x6400 + (code + 128) is 1152 + code in fp16
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
    uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 ha = __hsub2(*reinterpret_cast<__half2*>(&a), off);
    const __half2 hb = __hsub2(*reinterpret_cast<__half2*>(&b), off);
    h01 = *reinterpret_cast<const uint32_t*>(&ha);
    h23 = *reinterpret_cast<const uint32_t*>(&hb);
  } else {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
        " cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(h01), "=r"(h23)
        : "r"(w));
  }
}

// Query row `col` of the columns of a job.
struct Column {
  int seq, token, head;  // head: within the kv head's group
};
__device__ __forceinline__ Column column_of(const Plan& p, int seq, int col) {
  const int b = seq < 0 ? p.by_rows.of(col) : seq, r = seq < 0 ? col - b * p.rows : col;
  const int token = p.by_group.of(r);
  return {b, token, r - token * p.group};
}

// 16 values at p + i, in 16-byte loads where `vec` says that they are aligned.
template <int DT>
__device__ __forceinline__ void load16(const void* p, long long i, bool vec, float* x) {
  constexpr int N = Wide<DT>::kVals;
#pragma unroll
  for (int j = 0; j < 16 / N; ++j) {
    if (vec)
      load_vals<DT, true>(p, i + j * N, x + j * N);
    else
      load_vals<DT, false>(p, i + j * N, x + j * N);
  }
}

template <typename F>
inline void kvq_dispatch(int dtype, int format, int head_dim, bool vec, F&& f) {
  auto with_d = [&](auto dt, auto fmt) {
    auto with_vec = [&](auto d) {
      if (vec)
        f(dt, fmt, d, std::true_type{});
      else
        f(dt, fmt, d, std::false_type{});
    };
    if (head_dim == 64)
      with_vec(std::integral_constant<int, 64>{});
    else
      with_vec(std::integral_constant<int, 128>{});
  };
  auto with_fmt = [&](auto dt) {
    if (format == kKvqInt8)
      with_d(dt, std::integral_constant<int, kKvqInt8>{});
    else
      with_d(dt, std::integral_constant<int, kKvqE4m3>{});
  };
  if (dtype == kDtBf16)
    with_fmt(std::integral_constant<int, kDtBf16>{});
  else
    with_fmt(std::integral_constant<int, kDtF32>{});
}

// Whether every row of k and v starts on 16 bytes.
inline bool rows_aligned(const void* k, const void* v, int dtype, long long ks, long long vs) {
  const int n = dtype == kDtBf16 ? 8 : 4;
  return ks % n == 0 && vs % n == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(v) % 16 == 0;
}

// The shared pages on tcgen05 (kv_shared.cu): bf16 rows, p.tc_jobs > 0.
cudaError_t launch_shared(const KvqCache& c, const KvqAttention& a, const Plan& p, cudaStream_t s);

}  // namespace kvq
}  // namespace orx
