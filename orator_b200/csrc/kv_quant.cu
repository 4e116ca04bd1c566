// The 8-bit paged KV cache: quantising rows as they are written and reading
// them back. (Attention over it: kv_attention.cu, kv_shared.cu.)
//
// One (page, kv head) block, 16 tokens, D values each, is contiguous:
//   K codes [16][D] | V codes [16][D] | K scales [16] fp32 | V scales [16] fp32
// so one bulk copy brings all a head needs of a page. value = code * scale;
// per (token, head) row x: a = max|x|, scale = a / 127 (int8) or a / 448
// (e4m3) and code = RN(x / scale), each division correctly rounded in fp32,
// so the codes are a function of the row alone. A scale below the least
// normal number is stored as 0 with codes 0; a row with an infinity or a NaN
// gets a NaN scale and codes 0, and poisons what reads it, and only that.
#include "kv_quant.cuh"

namespace orx {
using namespace kvq;
namespace {

// Block of head 0 of position `pos` of sequence `seq`, or nullptr where the
// position or its page is outside the table or the pool (noted in *err);
// pos < 0: a padding row, skipped.
__device__ __forceinline__ uint8_t* block_of(const KvqCache& c, int seq, int pos) {
  if (pos < 0) return nullptr;
  const int j = pos / kPage;
  if (seq < 0 || seq >= c.seqs || j >= c.max_pages) {
    note_bad(c.err);
    return nullptr;
  }
  const int page = c.page_table[static_cast<long long>(seq) * c.max_pages + j];
  if (page < 0 || page >= c.pages) {
    note_bad(c.err);
    return nullptr;
  }
  return c.pool + static_cast<long long>(page) * c.kv_heads * kvq_block_bytes(c.head_dim);
}

// ---- writing and reading rows ---------------------------------------------
// A warp takes a run of units -- one (head, K or V) of D values each -- of one
// row, whose block is looked up once. A unit is the work of a few neighbouring
// lanes, which move its row in 16-byte pieces (4 fp32 or 8 bf16 values), and
// the loads of several units are under way together.
// a / kLimit, correctly rounded, for a >= 0 and a normal quotient: a quotient
// from the rounded reciprocal is within an ulp, and one step with its exact
// remainder then rounds as the division does (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990).
template <int FMT>
__device__ __forceinline__ float over_limit(float a) {
  constexpr float kLimit = FMT == kKvqInt8 ? 127.0f : 448.0f, kInv = 1.0f / kLimit;
  const float q = a * kInv;
  return fmaf(fmaf(-q, kLimit, a), kInv, q);
}

// Codes of 4 values x / s, each quotient correctly rounded before it is
// rounded to a code. x * (1 / s) is within 2^-22 of the quotient, so where the
// two ends of a band of 2^-21 around it round to the same code, that is the
// code; a value nearer to the middle between two codes (1 in 10^4) divides.
// lo, hi: 1 / s less and more 2^-21 (0 where all codes are 0). int8: adding
// 1.5 * 2^23 rounds to an integer, ties to even, and leaves it in the sum's low
// byte.
template <int FMT>
__device__ __forceinline__ uint32_t quantise4(const float* x, float s, float lo, float hi) {
  const float2 x0 = make_float2(x[0], x[1]), x1 = make_float2(x[2], x[3]);
  const float2 lo2 = make_float2(lo, lo), hi2 = make_float2(hi, hi);
  if (FMT == kKvqInt8) {
    constexpr float kMagic = 12582912.0f;
    const float2 m2 = make_float2(kMagic, kMagic);
    float2 a0 = fma2(x0, lo2, m2), a1 = fma2(x1, lo2, m2);
    const float2 b0 = fma2(x0, hi2, m2), b1 = fma2(x1, hi2, m2);
    if (a0.x != b0.x || a0.y != b0.y || a1.x != b1.x || a1.y != b1.y) {
      if (lo > 0.f) {
        a0 = make_float2(__fdiv_rn(x[0], s) + kMagic, __fdiv_rn(x[1], s) + kMagic);
        a1 = make_float2(__fdiv_rn(x[2], s) + kMagic, __fdiv_rn(x[3], s) + kMagic);
      }
    }
    return __byte_perm(__byte_perm(__float_as_uint(a0.x), __float_as_uint(a0.y), 0x0040),
                       __byte_perm(__float_as_uint(a1.x), __float_as_uint(a1.y), 0x0040), 0x5410);
  }
  auto pack = [](float2 a, float2 b) {
    const uint32_t p = __nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3);
    return p | static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3)) << 16;
  };
  const uint32_t w = pack(mul2(x0, lo2), mul2(x1, lo2));
  if (w == pack(mul2(x0, hi2), mul2(x1, hi2)) || !(lo > 0.f)) return w;
  return pack(make_float2(__fdiv_rn(x[0], s), __fdiv_rn(x[1], s)),
              make_float2(__fdiv_rn(x[2], s), __fdiv_rn(x[3], s)));
}

// Values of the N codes of w (4 a word) times s, rounded once. int8: the code
// with its sign bit flipped, as the low byte of 2^23, is 2^23 + 128 + code.
// e4m3: exact in fp16, where its NaN is one too.
template <int FMT, int N>
__device__ __forceinline__ void dequantise(const uint32_t* w, float s, float* x) {
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    if (FMT == kKvqInt8) {
      const uint32_t u = w[i] ^ 0x80808080u;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        x[4 * i + j] =
            (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440 + j)) - 8388736.0f) * s;
    } else {
      uint32_t h[2];
      codes_to_half<FMT>(w[i], h[0], h[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 f = unpack_half(h[j]);
        x[4 * i + 2 * j] = f.x * s;
        x[4 * i + 2 * j + 1] = f.y * s;
      }
    }
  }
}

constexpr int kUnroll = 4;

// The words of N codes.
template <int N>
__device__ __forceinline__ void read_codes(const uint8_t* src, uint32_t* w) {
  if (N == 8) {
    const uint2 t = *reinterpret_cast<const uint2*>(src);
    w[0] = t.x;
    w[N / 4 - 1] = t.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(src);
  }
}
// N values to p + i: 16 bytes, in one store where they are aligned.
template <int DT, bool VEC, int N>
__device__ __forceinline__ void store_vals(void* p, long long i, const float* x) {
  if (!VEC) {
#pragma unroll
    for (int j = 0; j < N; ++j) store_f(p, DT, i + j, x[j]);
  } else if (DT == kDtBf16) {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) =
        make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[N - 4], x[N - 3]),
                   pack_bf16(x[N - 2], x[N - 1]));
  } else {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// Writing: 16 values a lane (D / 16 lanes a unit), in 2 or 4 loads that are
// whole lines of the unit, so a scale costs few shuffles. The next step's loads
// are under way while a step is worked on. PACK: rows of few units, several
// side by side in the lanes (run_units units each, `runs` rows a warp), which
// would stand idle otherwise: 144,000 rows of one head of 64 values 62 us with
// a warp a row and 22 with one for four.
template <int DT, int FMT, int D, bool VEC, bool PACK>
__global__ void __launch_bounds__(256, 5) kvq_write_kernel(KvqCache c, const void* k, const void* v,
                                                        long long ks, long long vs,
                                                        const int* row_seq, const int* row_pos,
                                                        int rows, int runs, int run_units) {
  constexpr int N = Wide<DT>::kVals, kLoads = 16 / N, kLanes = D / 16, kStep = 32 / kLanes;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int part = lane % kLanes, slot = lane / kLanes;
  const int units = 2 * c.kv_heads;
  const int own = PACK ? slot / units : 0, mine = slot - own * units;  // the lane's row of the warp's, and unit
  if ((PACK ? w * runs : w / runs) >= rows) return;
  const int row = PACK ? min(w * runs + own, rows - 1) : w / runs;
  const int u0 = PACK ? 0 : (w - row * runs) * run_units;
  const int u1 = min(units, u0 + run_units);
  const int pos = row_pos[row];
  uint4 next[kLoads];
  auto load = [&](int u) {
    const int un = min(u + mine, u1 - 1);
    const long long off = static_cast<long long>(row) * (un & 1 ? vs : ks) + (un >> 1) * D + part * N;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      next[j] = load_raw<DT, VEC>(un & 1 ? v : k, off + j * kLanes * N);
  };
  if (u0 < u1) load(u0);
  uint8_t* b = nullptr;
  if (!PACK || (own < runs && w * runs + own < rows)) b = block_of(c, row_seq[row], pos);
  if (!PACK && !b) return;
  for (int u = u0; u < u1; u += kStep) {
    float x[16];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) unpack_raw<DT>(next[j], x + j * N);
    if (u + kStep < u1) load(u + kStep);
    const int un = u + mine;
    float top = 0.f;  // NaN where there is one
#pragma unroll
    for (int j = 0; j < 16; ++j)
      asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x[j])));
    uint32_t amax = __float_as_uint(top);  // ordered, infinities and NaN above every number
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1)
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float s = over_limit<FMT>(__uint_as_float(amax)), inv;
    if (s < 1.17549435e-38f) s = 0.f;
    if (amax >= 0x7f800000u) s = NAN;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
    if (!(s > 0.f)) inv = 0.f;
    const float lo = inv * (1.0f - 0x1p-21f), hi = inv * (1.0f + 0x1p-21f);
    uint32_t code[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      code[j] = quantise4<FMT>(x + 4 * j, s, lo, hi);
      if (!(s > 0.f)) code[j] = 0;  // and not 0 * infinity
    }
    if (un >= u1 || (PACK && !b)) continue;
    uint8_t* blk = b + (un >> 1) * kvq_block_bytes(D);
    const int at = (un & 1) * kPage + pos % kPage;
    uint8_t* dst = blk + at * D + part * N;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      if (N == 8)
        *reinterpret_cast<uint2*>(dst + j * kLanes * N) = make_uint2(code[2 * j % 4], code[(2 * j + 1) % 4]);
      else
        *reinterpret_cast<uint32_t*>(dst + j * kLanes * N) = code[j % 4];
    }
    if (part == 0) reinterpret_cast<float*>(blk + 2 * kPage * D)[at] = s;
  }
}

// Reading. PACK: rows of few units in a long call; a warp's kUnroll steps are
// `runs` rows of run_units units (144,000 rows of one head of 64 values 57 us
// with a warp a row, 17 with one for eight).
template <int DT, int FMT, int D, bool VEC, bool PACK>
__global__ void __launch_bounds__(256) kvq_read_kernel(KvqCache c, void* k, void* v, long long ks,
                                                       long long vs, const int* row_seq,
                                                       const int* row_pos, int rows, int runs,
                                                       int run_units) {
  constexpr int N = Wide<DT>::kVals, kLanes = D / N, kStep = 32 / kLanes;
  const int w = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int part = (lane % kLanes) * N;
  if constexpr (PACK) {
    const int first = w * runs, units = run_units;
    if (first >= rows) return;
    const uint8_t* blk[kUnroll];
    long long off[kUnroll];
    int at[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int slot = i * kStep + lane / kLanes, own = slot / units, un = slot - own * units;
      const int row = first + own;
      blk[i] = nullptr;
      if (own < runs && row < rows) {
        const int pos = row_pos[row];
        blk[i] = block_of(c, row_seq[row], pos);
        if (blk[i]) blk[i] += static_cast<long long>(un >> 1) * kvq_block_bytes(D);
        at[i] = (un & 1) * kPage + pos % kPage;
        off[i] = static_cast<long long>(row) * (un & 1 ? vs : ks) + (un >> 1) * D + part;
      }
    }
    uint32_t code[kUnroll][N / 4];
    float s[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (!blk[i]) continue;
      read_codes<N>(blk[i] + at[i] * D + part, code[i]);
      s[i] = reinterpret_cast<const float*>(blk[i] + 2 * kPage * D)[at[i]];
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      if (!blk[i]) continue;
      float x[N];
      dequantise<FMT, N>(code[i], s[i], x);
      store_vals<DT, VEC, N>(at[i] >= kPage ? v : k, off[i], x);
    }
    return;
  }
  const int row = w / runs;
  if (row >= rows) return;
  const int units = 2 * c.kv_heads, u0 = (w - row * runs) * run_units;
  const int u1 = min(units, u0 + run_units);
  const int pos = row_pos[row];
  const uint8_t* b = block_of(c, row_seq[row], pos);
  if (!b) return;
  for (int u = u0; u < u1; u += kUnroll * kStep) {
    uint32_t code[kUnroll][N / 4];
    float s[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int un = min(u + i * kStep + lane / kLanes, u1 - 1);
      const uint8_t* blk = b + static_cast<long long>(un >> 1) * kvq_block_bytes(D);
      const int at = (un & 1) * kPage + pos % kPage;
      read_codes<N>(blk + at * D + part, code[i]);
      s[i] = reinterpret_cast<const float*>(blk + 2 * kPage * D)[at];
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
      const int un = u + i * kStep + lane / kLanes;
      if (un >= u1) continue;
      float x[N];
      dequantise<FMT, N>(code[i], s[i], x);
      void* dst = un & 1 ? v : k;
      const long long off =
          static_cast<long long>(row) * (un & 1 ? vs : ks) + (un >> 1) * D + part;
      store_vals<DT, VEC, N>(dst, off, x);
    }
  }
}

// How a row's 2 * kv_heads units are cut into runs, one warp each. A warp of
// a long call takes kUnroll steps or more, so that the row's look-up is paid
// once; a short call (fewer warps than the GPU holds) is cut into single
// steps, where latency counts: 64 rows of 8 heads of 128.
struct Runs {
  int runs, units;
};
Runs row_runs(int rows, int kv_heads, int step) {
  const int units = 2 * kv_heads;
  int run = step;
  while (run < units && static_cast<long long>(rows) * ((units + run - 1) / run) > 148 * 16)
    run *= 2;
  return {(units + run - 1) / run, run};
}

}  // namespace

void op_kvq_write(const KvqCache& c, const void* k, const void* v, int dtype, long long ks,
                  long long vs, const int* row_seq, const int* row_pos, int rows, cudaStream_t s) {
  kvq_dispatch(dtype, c.format, c.head_dim, rows_aligned(k, v, dtype, ks, vs),
               [&](auto dt, auto fmt, auto d, auto vec) {
                 constexpr int kStep = 32 / (d / 16);
                 const int side = kStep / (2 * c.kv_heads);  // rows side by side
                 if (side > 1) {
                   const int warps = (rows + side - 1) / side;
                   kvq_write_kernel<dt, fmt, d, vec, true><<<(warps + 7) / 8, 256, 0, s>>>(
                       c, k, v, ks, vs, row_seq, row_pos, rows, side, 2 * c.kv_heads);
                   return;
                 }
                 const Runs r = row_runs(rows, c.kv_heads, kStep);
                 const long long warps = static_cast<long long>(rows) * r.runs;
                 kvq_write_kernel<dt, fmt, d, vec, false><<<static_cast<unsigned>((warps + 7) / 8), 256, 0, s>>>(
                     c, k, v, ks, vs, row_seq, row_pos, rows, r.runs, r.units);
               });
}

void op_kvq_read(const KvqCache& c, void* k, void* v, int dtype, long long ks, long long vs,
                 const int* row_seq, const int* row_pos, int rows, cudaStream_t s) {
  kvq_dispatch(dtype, c.format, c.head_dim, rows_aligned(k, v, dtype, ks, vs),
               [&](auto dt, auto fmt, auto d, auto vec) {
                 constexpr int kStep = 32 / (d / Wide<dt>::kVals);
                 const int units = 2 * c.kv_heads, side = kUnroll * kStep / units;
                 if (side > 1 && rows > 148 * 16) {
                   const int warps = (rows + side - 1) / side;
                   kvq_read_kernel<dt, fmt, d, vec, true><<<(warps + 7) / 8, 256, 0, s>>>(
                       c, k, v, ks, vs, row_seq, row_pos, rows, side, units);
                   return;
                 }
                 const Runs r = row_runs(rows, c.kv_heads, kStep);
                 const long long warps = static_cast<long long>(rows) * r.runs;
                 kvq_read_kernel<dt, fmt, d, vec, false><<<static_cast<unsigned>((warps + 7) / 8), 256, 0, s>>>(
                     c, k, v, ks, vs, row_seq, row_pos, rows, r.runs, r.units);
               });
}

}  // namespace orx
