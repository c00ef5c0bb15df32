// Linear of a few tokens over int4 weights with 16-bit activations, and its gated form.
//
//   y[m, n] = sum_g s[g, n] * sum_{k in group g} x[m, k] * c[n, k]        (one scale a row: s[n] * sum_k ...)
//   gated:    h[m, n] = silu(y[m, n]) * y[m, N + n]                       (weight rows [0, N) gate, [N, 2 N) up)
//
// Bound: the weights' bytes, read once.  Half a byte gives 2 M operations, so tensor instructions fed from registers are fast
// enough (mma.sync; a tcgen05 tile would be padding at these M and would want the expanded codes in shared memory first), and what
// counts is the bytes in flight.  A warp takes 16 MT weight rows and one 128-code unit a step: a unit's 16 rows are
// 1 KB in one piece, a lane holds 32 codes of two rows as two 16-byte loads, DEPTH units are on their way before the first is
// used, and the stream runs on over the block's row tiles without a break.  The tokens stay in shared memory, laid out once as
// the instruction's operand.
//
// Codes become exact 16-bit numbers without a conversion: a nibble, its top bit flipped, is or-ed (in one instruction with the
// mask) under the exponent of 128 (bf16) or 1024 (fp16), and one subtraction takes that off again.  The k order inside an
// instruction is free as long as both operands agree: a word's nibbles come out as pairs (i, i + 4), and the tokens are
// laid out in these pairs.  Products of a code and a 16-bit number are exact in fp32 and all sums are fp32; the result is rounded once.
//
// The eight warps of a block take every eighth unit and are added in ascending order through shared memory.  Where the tokens do
// not fit a block's shared memory, a cluster of 2 to 8 blocks splits K, and its ranks are added in order through
// distributed shared memory: no workspace, and the same bits in every run.
#include "common.cuh"
#include "ptx.cuh"
#include <type_traits>

namespace i4tc {

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr int kMostTokens = 32;                  // of a launch's grid row; more tokens read the weights again
constexpr size_t kMostSmem = 220 * 1024;

struct W4A16Params {
  const void* x;
  const uint8_t* w;
  const float* sw;      // [units, rows], or [rows]
  void* out;            // [M, N]
  long long ldx;
  int M, N, K;
  int rows;             // of the weights: N, gated 2 N
  int units;            // ceil(K / 128)
  int units_each;       // of a cluster rank
  int ranks;            // blocks of a cluster
  int tiles;            // of 16 MT weight rows (gated: 16 columns)
  int most_tokens;      // of a grid row
};

template <typename T>
__device__ __forceinline__ uint32_t codes_pair(uint32_t w) {   // nibbles 0 and 4 of w as two numbers of type T
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const uint32_t u = (w & 0x000F000Fu) ^ 0x43084308u;        // 128 + (code + 8)
    const uint32_t o = 0x43084308u;                             // 136
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&o));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const uint32_t u = (w & 0x000F000Fu) ^ 0x64086408u;        // 1024 + (code + 8)
    const uint32_t o = 0x64086408u;                             // 1032
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&o));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

__device__ __forceinline__ uint4 load_stream(const uint8_t* p) {   // read once: not kept in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }

// Floats of one warp's partial sums: rows padded so that the lanes of a fragment hit different banks.
__host__ __device__ constexpr int red_row(int mt) { return 16 * mt + 4; }
__host__ __device__ constexpr size_t w4a16_smem(int tokens, int units_each, int mt, int ranks) {
  return (size_t)units_each * tokens * 256                                // the tokens
         + (size_t)kWarps * tokens * red_row(mt) * 4                      // partial sums of the warps
         + (size_t)2 * (ranks - 1) * tokens * 16 * mt * 4;                // and of the other ranks, two tiles' worth
}

// NT: 8-token tiles.  MT: 16-row tiles of a warp (gated: one of gate rows, one of up rows).  ROWMAJOR: codes [rows, K / 2] and one
// scale a row, else [units, rows, 64] and a scale for each unit.
template <typename T, int NT, int MT, bool GATED, bool ROWMAJOR, int DEPTH>
__global__ void __launch_bounds__(kThreads) w4a16_kernel(const W4A16Params p) {
  static_assert(!GATED || MT == 2, "gate and up");
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.y, u0 = rank * p.units_each;
  const int units = min(p.units_each, p.units - u0);
  const int m0 = blockIdx.z * p.most_tokens, M = min(p.most_tokens, p.M - m0);
  uint4* xs = reinterpret_cast<uint4*>(smem);                             // [unit][word][token][t]
  float* red = reinterpret_cast<float*>(smem + (size_t)p.units_each * M * 256);   // [warp][token][row]
  float* other = red + kWarps * M * red_row(MT);                          // [parity][rank - 1][token][row]

  const T* x = pdl_wait(static_cast<const T*>(p.x));
  const uint8_t* w = p.w;
  const float* sw = p.sw;
  pdl_fresh(w); pdl_fresh(sw);

  const int steps = (units + kWarps - 1) / kWarps;                        // of a row tile; the same for every warp
  uint4 ring[DEPTH][MT][2];
  float scale[DEPTH][MT][2];
  int f_tile = blockIdx.x, f_step = 0;                                    // where the loads are
  // Rows behind the last read the last row (their sums go nowhere); units behind the last are zero codes.
  auto fetch = [&](uint4 (&v)[MT][2], float (&s)[MT][2]) {
    const int u = f_step * kWarps + warp;
    if (f_tile < p.tiles && u < units) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int r = (GATED ? f_tile * 16 : f_tile * 16 * MT + 16 * mt) + g + 8 * h;
          r = min(r, p.N - 1) + (GATED && mt == 1 ? p.N : 0);
          if constexpr (ROWMAJOR) {
            const int k = (u0 + u) * 128 + t * 32;
            v[mt][h] = make_uint4(0u, 0u, 0u, 0u);
            if (k < p.K) v[mt][h] = load_stream(w + (long long)r * (p.K / 2) + k / 2);
          } else {
            const long long at = (long long)(u0 + u) * p.rows + r;
            v[mt][h] = load_stream(w + at * 64 + t * 16);
            s[mt][h] = __ldg(sw + at);
          }
        }
      }
    }
    if (++f_step == steps) { f_step = 0; f_tile += gridDim.x; }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) fetch(ring[d], scale[d]);

  // the tokens, as the operand of the instruction: 16 bytes = eight numbers of one token in pairs (i, i + 4)
  for (int i = threadIdx.x; i < units * 16 * M; i += kThreads) {
    const int m = i / (units * 16), c = i - m * (units * 16), k = u0 * 128 + c * 8;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (k < p.K) v = __ldg(reinterpret_cast<const uint4*>(x + (long long)(m0 + m) * p.ldx + k));
    xs[(((c >> 4) * 4 + (c & 3)) * M + m) * 4 + ((c >> 2) & 3)] =
        make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
  }
  if (p.ranks > 1) ptx::cluster_sync(); else __syncthreads();

  float f[MT][NT][4];
  int tile = blockIdx.x, step = 0, parity = 0;
  auto clear = [&](float (&a)[MT][NT][4]) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) a[mt][nt][i] = 0.f;
  };
  auto multiply = [&](const uint4 (&v)[MT][2], int u, float (&c)[MT][NT][4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint4 b[NT];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        b[nt] = make_uint4(0u, 0u, 0u, 0u);
        if (8 * nt + g < M) b[nt] = xs[((u * 4 + q) * M + 8 * nt + g) * 4 + t];
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const uint32_t a = q == 0 ? v[mt][0].x : q == 1 ? v[mt][0].y : q == 2 ? v[mt][0].z : v[mt][0].w;
        const uint32_t e = q == 0 ? v[mt][1].x : q == 1 ? v[mt][1].y : q == 2 ? v[mt][1].z : v[mt][1].w;
        const uint32_t a0 = codes_pair<T>(a), a1 = codes_pair<T>(a >> 4), a2 = codes_pair<T>(a >> 8), a3 = codes_pair<T>(a >> 12);
        const uint32_t e0 = codes_pair<T>(e), e1 = codes_pair<T>(e >> 4), e2 = codes_pair<T>(e >> 8), e3 = codes_pair<T>(e >> 12);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16<T>(c[mt][nt], a0, e0, a1, e1, b[nt].x, b[nt].y);
          mma16<T>(c[mt][nt], a2, e2, a3, e3, b[nt].z, b[nt].w);
        }
      }
    }
  };
  // The tile's sums, warp by warp and rank by rank in ascending order; every thread of the block (of the cluster) comes here.
  auto finish = [&]() {
    float* mine = red + warp * M * red_row(MT);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int m = 8 * nt + 2 * t + (i & 1);
          if (m < M) mine[m * red_row(MT) + 16 * mt + g + 8 * (i >> 1)] = f[mt][nt][i];
        }
    __syncthreads();
    auto sum = [&](int m, int r) {
      float v = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v += red[(k * M + m) * red_row(MT) + r];
      return v;
    };
    const int values = M * 16 * MT;
    if (p.ranks > 1) {
      if (rank > 0) {
        const uint32_t to = ptx::mapa_shared(ptx::smem_u32(other + (parity * (p.ranks - 1) + rank - 1) * values), 0);
        for (int i = threadIdx.x; i < values; i += kThreads) {
          const int m = i / (16 * MT), r = i - m * (16 * MT);
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(to + 4u * i), "f"(sum(m, r)) : "memory");
        }
      }
      ptx::cluster_sync();
    }
    if (rank == 0) {
      const float* more = other + parity * (p.ranks - 1) * values;
      auto total = [&](int m, int r) {
        float v = sum(m, r);
        for (int k = 0; k + 1 < p.ranks; ++k) v += more[(k * M + m) * (16 * MT) + r];
        return v;
      };
      constexpr int COLS = GATED ? 16 : 16 * MT;
      for (int i = threadIdx.x; i < M * COLS; i += kThreads) {
        const int m = i / COLS, r = i - m * COLS, n = tile * COLS + r;
        if (n >= p.N) continue;
        float v = total(m, r);
        if constexpr (ROWMAJOR) v *= __ldg(sw + n);
        if constexpr (GATED) {
          float up = total(m, r + 16);
          if constexpr (ROWMAJOR) up *= __ldg(sw + p.N + n);
          v = v / (1.0f + expf(-v)) * up;
        }
        store_as(static_cast<T*>(p.out) + (long long)(m0 + m) * p.N + n, v);
      }
    }
    __syncthreads();
  };

  clear(f);
  while (tile < p.tiles) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      if (tile < p.tiles) {
        const int u = step * kWarps + warp;
        if (u < units) {
          if constexpr (ROWMAJOR) {
            multiply(ring[d], u, f);
          } else {
            float c[MT][NT][4];
            clear(c);
            multiply(ring[d], u, c);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) f[mt][nt][i] = fmaf(c[mt][nt][i], scale[d][mt][i >> 1], f[mt][nt][i]);
          }
        }
        fetch(ring[d], scale[d]);
        if (++step == steps) {
          finish();
          clear(f);
          step = 0;
          parity ^= 1;
          tile += gridDim.x;
        }
      }
    }
  }
}

template <typename T, int NT, int MT, bool GATED, bool ROWMAJOR>
int launch_one(const W4A16Params& p, dim3 grid, size_t smem, cudaStream_t st) {
  constexpr int DEPTH = MT == 2 ? 3 : 4;
  auto kernel = w4a16_kernel<T, NT, MT, GATED, ROWMAJOR, DEPTH>;
  // the limit belongs to the function, not to a launch: set once, to the most that any call asks for
  static bool configured[64] = {false};
  int dev = 0;
  I4TC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    I4TC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostSmem));
    if (dev < 64) configured[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 1;
  attr[1].val.clusterDim.y = (unsigned)p.ranks;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.ranks > 1 ? 2 : 1;
  I4TC_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  return I4TC_OK;
}

template <typename T, bool GATED, bool ROWMAJOR>
int launch_tokens(const W4A16Params& p, dim3 grid, size_t smem, cudaStream_t st) {
  const int m = p.M < p.most_tokens ? p.M : p.most_tokens;
  if (m <= 8) return launch_one<T, 1, 2, GATED, ROWMAJOR>(p, grid, smem, st);
  if (m <= 16) return launch_one<T, 2, 2, GATED, ROWMAJOR>(p, grid, smem, st);
  return launch_one<T, 4, 2, GATED, ROWMAJOR>(p, grid, smem, st);
}

}  // namespace

}  // namespace i4tc

using namespace i4tc;

extern "C" int i4tc_w4a16_linear(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const uint8_t* w, const float* w_scale,
                                 int per_channel, int gated, void* out, int64_t N, int device, void* stream) {
  I4TC_REQUIRE(dtype == I4TC_BF16 || dtype == I4TC_FP16, I4TC_EUNSUPPORTED, "activations must be bfloat16 or float16");
  I4TC_REQUIRE(M >= 0 && N >= 0 && K > 0, I4TC_EINVAL, "bad size");
  if (M == 0 || N == 0) return I4TC_OK;
  I4TC_REQUIRE(x && w && w_scale && out, I4TC_EINVAL, "null pointer");
  if (per_channel) {
    I4TC_REQUIRE(K % 64 == 0, I4TC_EINVAL, "K must be a multiple of 64");
  } else {
    I4TC_REQUIRE(K % 128 == 0, I4TC_EINVAL, "K must be divisible by group_size");
  }
  I4TC_REQUIRE(K <= (1 << 20) && N < (1ll << 29) && M < (1ll << 20), I4TC_EINVAL, "operand too large");
  I4TC_REQUIRE(aligned_to(x, 16) && aligned_to(w, 16) && ldx % 8 == 0 && aligned_to(w_scale, 4), I4TC_EALIGN,
               "activations and weights must be 16-byte aligned");
  const DeviceInfo* info;
  if (int rc = device_info(device, &info)) return rc;
  I4TC_REQUIRE(info->cc_major == 10, I4TC_EDEVICE, "device %d is sm_%d%d; this library needs sm_100", device, info->cc_major, info->cc_minor);
  DeviceGuard guard(device);
  I4TC_CUDA(guard.err);
  W4A16Params p = {};
  p.x = x; p.w = w; p.sw = w_scale; p.out = out; p.ldx = ldx;
  p.M = (int)M; p.N = (int)N; p.K = (int)K;
  p.rows = gated ? 2 * p.N : p.N;
  p.units = (p.K + 127) / 128;
  p.tiles = (p.N + (gated ? 15 : 31)) / (gated ? 16 : 32);
  // as many tokens at a time, up to 32, as a cluster of eight blocks has room for
  p.most_tokens = kMostTokens;
  while (p.most_tokens > 1 && w4a16_smem(p.most_tokens < p.M ? p.most_tokens : p.M, (p.units + 7) / 8, 2, 8) > kMostSmem) p.most_tokens /= 2;
  const int tokens = p.M < p.most_tokens ? p.M : p.most_tokens;
  // K in one block where two blocks' tokens fit an SM, else over the smallest cluster where they do
  p.ranks = 1;
  while (p.ranks < 8 && p.ranks * 2 <= p.units && w4a16_smem(tokens, (p.units + p.ranks - 1) / p.ranks, 2, p.ranks) > kMostSmem / 2) p.ranks *= 2;
  p.units_each = (p.units + p.ranks - 1) / p.ranks;
  while (p.ranks > 1 && (p.ranks - 1) * p.units_each >= p.units) p.ranks /= 2, p.units_each = (p.units + p.ranks - 1) / p.ranks;
  const size_t smem = w4a16_smem(tokens, p.units_each, 2, p.ranks);
  I4TC_REQUIRE(smem <= kMostSmem, I4TC_EUNSUPPORTED, "K is too large");
  const int slots = info->sm_count * (smem > kMostSmem / 2 ? 1 : 2) / p.ranks;
  const dim3 grid((unsigned)(p.tiles < slots ? p.tiles : slots), (unsigned)p.ranks, (unsigned)((p.M + p.most_tokens - 1) / p.most_tokens));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto pick = [&](auto type) {
    using T = decltype(type);
    return gated ? (per_channel ? launch_tokens<T, true, true>(p, grid, smem, st) : launch_tokens<T, true, false>(p, grid, smem, st))
                 : (per_channel ? launch_tokens<T, false, true>(p, grid, smem, st) : launch_tokens<T, false, false>(p, grid, smem, st));
  };
  return dtype == I4TC_BF16 ? pick(__nv_bfloat16{}) : pick(__half{});
}
