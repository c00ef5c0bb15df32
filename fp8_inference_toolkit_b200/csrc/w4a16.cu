// Linear of a few tokens over int4 weights with 16-bit activations, and its gated form.
//
//   y[m, n] = sum_g s[g, n] * sum_{k in group g} x[m, k] * c[n, k]        (one scale a row: s[n] * sum_k ...)
//   gated:    h[m, n] = silu(y[m, n]) * y[m, N + n]                       (weight rows [0, N) gate, [N, 2 N) up)
//
// Bound: the weights' bytes, read once; then the instructions that a code costs.  Half a byte gives 2 M operations, so tensor
// instructions fed from registers are fast enough (mma.sync; a tcgen05 tile would be padding at these M and would want the expanded
// codes in shared memory first): an m16n8k16 takes a scheduler 8 cycles, and masking instructions run beside it.
//
// A block (sixteen warps, one an SM) takes a contiguous range of 16-row tiles, so that every SM has the same share whatever N is.
// Its warps take the tiles in turn, split K, or both.  A step is one tile's 128 codes of K (1 KB) and their scales, which a lane
// copies for itself into a ring of the warp's, up to eight steps ahead, by cp.async: no registers and no barrier, and no waiting on
// loads issued later (with the ring in registers the six scoreboards of a warp were shared between its steps, which cost the gated
// [1, 4096] x [24576, 4096] 4.6 us; bulk copies on mbarriers cost 80 instructions a step).
//
// Codes become operands of the tokens' type by masking and a subtraction: a nibble with its top bit flipped, in the low bits of the
// number 128 (bf16) or 1024 (fp16), is that number + 8 + code, and the difference is exact.  So are the products, and the fp32 sums hold
// nothing but the formula's terms: where a code is zero, the token's number has no part, however large.  (Leaving the +8 in and taking 8
// times the tokens' sum off the result saves the subtraction, 1.5 us of 16.4 for one gated token, but a number
// 2^20 times as large as the others then costs their sums 20 bits wherever its code is zero.)
//
// The k order inside an instruction is free as long as both operands agree: a word's nibbles come out as pairs (i, i + 4), and the
// tokens are laid out in these pairs, once, in shared memory.
//
// A cluster of up to eight blocks shares the same rows and splits K, where the tokens of long K would not fit a block, or where
// laying them out in every block costs more than adding up; its partial sums are added in ascending order through distributed
// shared memory: no workspace, no second launch, and the same bits in every run.
//
// Measured (device time, weights from HBM, bf16, per-group scales): [1, 4096] x [6144, 4096] 5.9 us, [16, 12288] x [4096, 12288]
// 14.4, gated [1, 4096] x [24576, 4096] 16.0 (3.3 TB/s), [16, ...] 20.9, [32, ...] 37.3.
#include "common.cuh"
#include "ptx.cuh"
#include <type_traits>

namespace i4tc {

namespace {

constexpr int kLogWarps = 4, kWarps = 1 << kLogWarps, kThreads = kWarps * 32;
constexpr int kMostTokens = 32;                     // of a launch's grid row; more tokens read the weights again
constexpr size_t kMostSmem = 224 * 1024;
constexpr int kStep = 16 * 64 + 16 * 4;             // bytes of a step: sixteen rows of 128 codes, and their scales

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
  int tiles;            // of sixteen weight rows
  int tile_warps;       // warps of a block that take its tiles in turn; the others split the block's K
  int steps;            // units of a warp, at most
  int most_tokens;      // of a grid row
};

// c = a b, or with ADD c += a b.
template <typename T, bool ADD>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  const float z[4] = {ADD ? c[0] : 0.f, ADD ? c[1] : 0.f, ADD ? c[2] : 0.f, ADD ? c[3] : 0.f};
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]));
  }
}

// 16 bytes global -> shared without registers in between; where not valid, nothing is read and zeros are written.
__device__ __forceinline__ void copy_16(uint32_t dst, const uint8_t* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16u : 0u) : "memory");
}
// (w & MASK) ^ flip in one instruction: one immediate operand, the other in a register that the compiler does not see through.
template <uint32_t MASK>
__device__ __forceinline__ uint32_t mask_flip(uint32_t w, uint32_t flip) {
  uint32_t u;
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(u) : "r"(w), "n"(MASK), "r"(flip));
  return u;
}
template <uint32_t V>
__device__ __forceinline__ uint32_t opaque() {
  uint32_t v;
  asm volatile("mov.u32 %0, %1;" : "=r"(v) : "n"(V));
  return v;
}

// Nibbles 0 and 4 of w as two numbers of type T.
template <typename T>
__device__ __forceinline__ uint32_t codes_pair(uint32_t w, uint32_t bias) {
  const uint32_t u = mask_flip<0x000F000Fu>(w, bias);
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), *reinterpret_cast<const __half2*>(&bias));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}

__device__ __forceinline__ void store_as(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_as(__half* p, float v) { *p = __float2half_rn(v); }

constexpr int token_tiles(int tokens, bool small) { return small || tokens > 24 ? 4 : (tokens + 7) / 8; }
constexpr int ring_depth(int token_tiles) { return token_tiles == 1 ? 8 : 4; }
constexpr size_t w4a16_smem(int tokens, bool small, int units_each, int block_tiles, int k_warps) {
  return (size_t)units_each * tokens * 256                              // the tokens
         + (size_t)block_tiles * k_warps * tokens * 64                  // partial sums
         + (size_t)kWarps * ring_depth(token_tiles(tokens, small)) * kStep;   // rings
}

// NT: 8-token tiles.  GATED: a tile's sixteen rows are eight columns' gate rows and then their up rows.  ROWMAJOR: codes [rows, K / 2]
// and one scale a row, else [units, rows, 64] and a scale for each unit.  SMALL: fewer columns than a tile has.
template <typename T, int NT, bool GATED, bool ROWMAJOR, bool SMALL>
__global__ void __launch_bounds__(kThreads, 1) w4a16_kernel(const W4A16Params p) {
  constexpr int COLS = GATED ? 8 : 16, DEPTH = ring_depth(NT);
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int rank = blockIdx.y, u0 = rank * p.units_each;
  const int units = min(p.units_each, p.units - u0);
  const int m0 = blockIdx.z * p.most_tokens, M = min(p.most_tokens, p.M - m0);
  const int tile0 = (int)((long long)blockIdx.x * p.tiles / gridDim.x), ntiles = (int)((long long)(blockIdx.x + 1) * p.tiles / gridDim.x) - tile0;
  const int wn = warp % p.tile_warps, wk = warp / p.tile_warps, k_warps = kWarps / p.tile_warps;
  const int first = min(units, wk * p.steps), mine = min(units, first + p.steps) - first;   // of the block's units, this warp's
  uint4* xs = reinterpret_cast<uint4*>(smem);                             // [unit][token][word][t], words of odd tokens swapped in pairs
  uint8_t* rings = reinterpret_cast<uint8_t*>(xs + (size_t)p.units_each * M * 16);   // [warp][slot][16 rows of codes, 16 scales]
  float* part = reinterpret_cast<float*>(rings + kWarps * DEPTH * kStep); // [tile][k warp][token][16]
  const uint32_t ring = ptx::smem_u32(rings) + warp * DEPTH * kStep, ring_lane = ring + lane * 16;

  const T* x = pdl_wait(static_cast<const T*>(p.x));
  const uint8_t* w = p.w;
  const float* sw = p.sw;
  pdl_fresh(w); pdl_fresh(sw);
  pdl_trigger();

  // The last tile begins early enough to be full: its first columns are the tile's before it, too, with the same bits.
  auto first_column = [&](int tile) -> long long { return SMALL ? 0 : min(tile * COLS, p.N - COLS); };
  // Row r of a tile, counted from its first column: rows behind the last read the last (their sums go nowhere).
  auto row_of = [&](int r) -> long long {
    const int c = GATED ? r & 7 : r;
    return (SMALL ? min(c, p.N - 1) : c) + (GATED && r >= 8 ? (long long)p.N : 0);
  };
  const int total = ntiles > wn && mine > 0 ? (ntiles - wn + p.tile_warps - 1) / p.tile_warps * mine : 0;   // steps of this warp
  // Where its copies are: lane (g, t) copies 32 codes each of rows g and 8 + g, for itself, and one of sixteen lanes a scale.
  const long long row_bytes = ROWMAJOR ? p.K / 2 : 64, unit_step = ROWMAJOR ? 64 : (long long)p.rows * 64;
  const uint8_t* const base_w = w + (ROWMAJOR ? (long long)(u0 + first) * 64 : (long long)(u0 + first) * p.rows * 64) + row_of(g) * row_bytes + t * 16;
  const float* const base_s = sw + (long long)(u0 + first) * p.rows + row_of(lane & 15);
  const long long second = row_of(8 + g) - row_of(g);
  const int lane_units = ROWMAJOR ? (p.K - (u0 + first) * 128 - t * 32 + 127) / 128 : 0;   // row-major: the last unit may be half
  int a_tile = tile0 + wn, a_u = 0;
  const uint8_t* a_w;
  const float* a_s;
  auto aim = [&]() {
    const long long row = first_column(a_tile);
    a_w = base_w + row * row_bytes;
    a_s = base_s + row;
  };
  auto fetch = [&](int slot) {
    const uint32_t to = ring_lane + slot * kStep;
    const bool in = !ROWMAJOR || a_u < lane_units;
    copy_16(to, in ? a_w : w, in);
    copy_16(to + 512, in ? a_w + second * row_bytes : w, in);
    if constexpr (!ROWMAJOR) {
      if (lane < 16) ptx::cp_async_4_zfill(ring + slot * kStep + 1024 + lane * 4, a_s, true);
      a_s += p.rows;
    }
    a_w += unit_step;
    if (++a_u == mine) {
      a_u = 0;
      a_tile += p.tile_warps;
      aim();                                                              // (an address only: behind the last tile nothing is read)
    }
  };
  aim();

  // The tokens, as the operand of the instruction: 16 bytes = eight numbers of one token in pairs (i, i + 4).  Sixteen lanes have a token's
  // numbers of a unit.  They are asked for before the weights, which all blocks ask for by the megabyte: behind those the sixteen tokens
  // of K 12288 came 4 us later.
  constexpr int BATCH = 8;                                                // passes whose loads are on their way together
  const int chunk = threadIdx.x & 15, passes = (units * M + kThreads / 16 - 1) / (kThreads / 16);
  struct Row {
    int u, m;
  };
  const int step_m = kThreads / 16 / units, step_u = kThreads / 16 - step_m * units;
  auto advance = [&](Row& r) {
    r.u += step_u;
    r.m += step_m;
    if (r.u >= units) { r.u -= units; ++r.m; }
  };
  auto load = [&](uint4 (&v)[BATCH], Row& at, int count) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      v[j] = make_uint4(0u, 0u, 0u, 0u);
      if (j >= count) continue;
      const int k = (u0 + at.u) * 128 + chunk * 8;
      if (at.m < M && k < p.K) v[j] = __ldg(reinterpret_cast<const uint4*>(x + (long long)(m0 + at.m) * p.ldx + k));
      advance(at);
    }
  };
  auto keep = [&](const uint4 (&v)[BATCH], Row& at, int count) {
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      if (j >= count) break;
      if (at.m < M)
        xs[(at.u * M + at.m) * 16 + ((chunk & 3) ^ (at.m & 1)) * 4 + (chunk >> 2)] = make_uint4(
            __byte_perm(v[j].x, v[j].z, 0x5410), __byte_perm(v[j].x, v[j].z, 0x7632), __byte_perm(v[j].y, v[j].w, 0x5410), __byte_perm(v[j].y, v[j].w, 0x7632));
      advance(at);
    }
  };
  uint4 held[BATCH];
  Row loaded = {(int)(threadIdx.x >> 4) % units, (int)(threadIdx.x >> 4) / units}, kept = loaded;
  int laid_out = 0;
#pragma unroll 1
  for (; laid_out + BATCH < passes; laid_out += BATCH) {
    load(held, loaded, BATCH);
    keep(held, kept, BATCH);
  }
  load(held, loaded, passes - laid_out);
#pragma unroll 1
  for (int d = 0; d < DEPTH; ++d) {
    if (d < total) fetch(d);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  keep(held, kept, passes - laid_out);
  __syncthreads();

  // a lane without a token of its own reads the last one: its column of the result goes nowhere
  uint32_t b_at[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int m = min(8 * nt + g, M - 1);
    b_at[nt] = ptx::smem_u32(xs) + (m * 16 + (m & 1) * 4 + t) * 16;
  }
  // 128 + 8 in bf16 or 1024 + 8 in fp16, twice
  const uint32_t bias = opaque<std::is_same_v<T, __nv_bfloat16> ? 0x43084308u : 0x64086408u>();
  float f[NT][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int i = 0; i < 4; ++i) f[nt][i] = 0.f;
  uint32_t b_off = first * M * 256;
  int u = 0, tile = wn;
  int slot = 0;
  for (int i = 0; i < total; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(DEPTH - 1) : "memory");
    __syncwarp();
    const uint32_t from = ring_lane + slot * kStep;
    const uint4 v0 = ptx::lds128(from), v1 = ptx::lds128(from + 512);
    float s0 = 1.0f, s1 = 1.0f;
    if constexpr (!ROWMAJOR) {
      const uint32_t s_from = ring + slot * kStep + 1024 + g * 4;
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s0) : "r"(s_from));
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(s1) : "r"(s_from + 32));
    }
    float c[NT][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t a[8];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4& v = h ? v1 : v0;
        const uint32_t word = q == 0 ? v.x : q == 1 ? v.y : q == 2 ? v.z : v.w;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[2 * k + h] = codes_pair<T>(word >> (4 * k), bias);
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint4 b = ptx::lds128(((b_at[nt] + b_off) ^ ((q & 1) * 64)) + (q >> 1) * 128);
        if (q == 0) mma16<T, false>(c[nt], a[0], a[1], a[2], a[3], b.x, b.y);
        else mma16<T, true>(c[nt], a[0], a[1], a[2], a[3], b.x, b.y);
        mma16<T, true>(c[nt], a[4], a[5], a[6], a[7], b.z, b.w);
      }
    }
    __syncwarp();                                                   // the slot has been read
    if (i + DEPTH < total) fetch(slot);
    asm volatile("cp.async.commit_group;" ::: "memory");
    if (++slot == DEPTH) slot = 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 4; ++j) f[nt][j] = fmaf(c[nt][j], j >> 1 ? s1 : s0, f[nt][j]);
    b_off += M * 256;
    if (++u == mine) {                                              // the tile's sums over this warp's units
      float* to = part + (tile * k_warps + wk) * M * 16;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int m = 8 * nt + 2 * t + (j & 1);
          if (m < M) to[m * 16 + g + 8 * (j >> 1)] = f[nt][j];
          f[nt][j] = 0.f;
        }
      u = 0;
      b_off = first * M * 256;
      tile += p.tile_warps;
    }
  }
  __syncthreads();

  // the warps' sums in ascending order (those that have units), then the ranks'
  const int with_work = min(k_warps, (units + p.steps - 1) / p.steps), values = ntiles * M * COLS;
  auto added = [&](int at) {
    float v = part[at];
    for (int k = 1; k < with_work; ++k) v += part[at + k * M * 16];
    return v;
  };
  auto finish = [&](int tile, int m, int r, float v, float up) {
    const long long n = first_column(tile0 + tile) + r;
    if (SMALL && n >= p.N) return;
    if constexpr (ROWMAJOR) v *= __ldg(sw + n);
    if constexpr (GATED) {
      if constexpr (ROWMAJOR) up *= __ldg(sw + p.N + n);
      v = v / (1.0f + expf(-v)) * up;
    }
    store_as(static_cast<T*>(p.out) + (long long)(m0 + m) * p.N + n, v);
  };
  if (p.ranks == 1) {
    for (int i = threadIdx.x; i < values; i += kThreads) {
      const int r = i % COLS, q = i / COLS, tile = q / M, m = q - tile * M, at = (tile * k_warps * M + m) * 16 + r;
      finish(tile, m, r, added(at), GATED ? added(at + 8) : 0.f);
    }
    return;
  }
  if (with_work > 1) {
    for (int i = threadIdx.x; i < ntiles * M * 16; i += kThreads) {
      const int q = i / 16, tile = q / M, at = (tile * k_warps * M + q - tile * M) * 16 + i % 16;
      part[at] = added(at);
    }
  }
  ptx::cluster_sync();
  // every rank adds an equal share of the values
  const int share = (values + p.ranks - 1) / p.ranks;
  const uint32_t base = ptx::smem_u32(part);
  for (int i = rank * share + threadIdx.x; i < min(values, (rank + 1) * share); i += kThreads) {
    const int r = i % COLS, q = i / COLS, tile = q / M, m = q - tile * M, at = (tile * k_warps * M + m) * 16 + r;
    float of[8], of_up[8];                                                // all on their way before the first is added
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      of[k] = of_up[k] = 0.f;
      if (k < p.ranks) {
        const uint32_t from = ptx::mapa_shared(base, k) + 4u * at;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(of[k]) : "r"(from));
        if constexpr (GATED) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(of_up[k]) : "r"(from + 32u));
      }
    }
    float v = 0.f, up = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v += of[k];
      up += of_up[k];
    }
    finish(tile, m, r, v, up);
  }
  ptx::cluster_sync();   // the others may still be reading
}

template <typename T, int NT, bool GATED, bool ROWMAJOR, bool SMALL>
int launch_one(const W4A16Params& p, dim3 grid, size_t smem, cudaStream_t st) {
  auto kernel = w4a16_kernel<T, NT, GATED, ROWMAJOR, SMALL>;
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

// Clusters of 1, 2, 4 and 8 blocks that run side by side, a block an SM (148, 74, 33 and 15 here: clusters do not cross a GPC).
int clusters_at_once(int device, const DeviceInfo* info, int (&out)[4]) {
  static std::atomic<int> known[64][4];
  for (int i = 0; i < 4; ++i) {
    out[i] = known[device][i].load();
    if (out[i] > 0) continue;
    if (i == 0) {
      out[i] = info->sm_count;
    } else {
      auto kernel = w4a16_kernel<__nv_bfloat16, 4, false, false, false>;
      I4TC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostSmem));
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(1u, 1u << i, 1);
      cfg.blockDim = dim3(kThreads, 1, 1);
      cfg.dynamicSmemBytes = kMostSmem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 1;
      attr.val.clusterDim.y = 1u << i;
      attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      I4TC_CUDA(cudaOccupancyMaxActiveClusters(&out[i], kernel, &cfg));
      if (out[i] < 1) out[i] = -1;   // this device holds none of that size
    }
    known[device][i].store(out[i]);
  }
  return I4TC_OK;
}

template <typename T, bool GATED, bool ROWMAJOR>
int launch_tokens(const W4A16Params& p, dim3 grid, size_t smem, cudaStream_t st) {
  if (p.N < (GATED ? 8 : 16)) return launch_one<T, 4, GATED, ROWMAJOR, true>(p, grid, smem, st);
  switch (token_tiles(p.M < p.most_tokens ? p.M : p.most_tokens, false)) {
    case 1: return launch_one<T, 1, GATED, ROWMAJOR, false>(p, grid, smem, st);
    case 2: return launch_one<T, 2, GATED, ROWMAJOR, false>(p, grid, smem, st);
    case 3: return launch_one<T, 3, GATED, ROWMAJOR, false>(p, grid, smem, st);
    default: return launch_one<T, 4, GATED, ROWMAJOR, false>(p, grid, smem, st);
  }
}

}  // namespace

}  // namespace i4tc

using namespace i4tc;

extern "C" int i4tc_w4a16_linear(const i4tc_w4a16_args* a, int device, void* stream) {
  I4TC_REQUIRE(a != nullptr, I4TC_EINVAL, "null pointer");
  const int64_t dtype = a->dtype, M = a->M, K = a->K, N = a->N, ldx = a->ldx;
  const void* x = a->x;
  const uint8_t* w = a->w;
  const float* w_scale = a->w_scale;
  void* out = a->out;
  const bool per_channel = a->per_channel != 0, gated = a->gated != 0;
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
  const int cols = gated ? 8 : 16;
  const bool small = p.N < cols;
  p.tiles = (p.N + cols - 1) / cols;
  // as many tokens at a time, up to 32, as a cluster of eight blocks has room for
  p.most_tokens = kMostTokens;
  while (p.most_tokens > 1 && w4a16_smem(p.most_tokens < p.M ? p.most_tokens : p.M, small, (p.units + 7) / 8, 2, 1) > kMostSmem) p.most_tokens /= 2;
  const int tokens = p.M < p.most_tokens ? p.M : p.most_tokens, chunks = (p.M + p.most_tokens - 1) / p.most_tokens;
  const int nt = token_tiles(tokens, small);
  double best = 0;
  int grid_x = 0;
  int at_once[4];
  if (int rc = clusters_at_once(device, info, at_once)) return rc;
  for (int i = 0; i < 4; ++i) {
    const int ranks = 1 << i;
    if (ranks > p.units || at_once[i] < 1) continue;
    const int each = (p.units + ranks - 1) / ranks;
    if ((ranks - 1) * each >= p.units) continue;
    const int most_x = at_once[i] > p.tiles ? p.tiles : at_once[i], most_tiles = (p.tiles + most_x - 1) / most_x;
    for (int j = 0; 1 << j <= kWarps; ++j) {   // (shifts: the way is chosen in every call, which waits for the host where it is short)
      const int tw = 1 << j, k_warps = kWarps >> j, steps = (each + k_warps - 1) >> (kLogWarps - j);
      // partial sums of all of a block's tiles have to fit: else more blocks, in waves
      int gx = most_x, block_tiles = most_tiles;
      while (block_tiles > 1 && w4a16_smem(tokens, small, each, block_tiles, k_warps) > kMostSmem) {
        gx *= 2;
        gx = gx > p.tiles ? p.tiles : gx;
        block_tiles = (p.tiles + gx - 1) / gx;
      }
      if (w4a16_smem(tokens, small, each, block_tiles, k_warps) > kMostSmem) continue;
      const int64_t blocks = (int64_t)gx * chunks, waves = blocks <= at_once[i] ? 1 : (blocks + at_once[i] - 1) / at_once[i];
      const int warp_steps = ((block_tiles + tw - 1) >> j) * steps;
      // Microseconds.  A warp scheduler (it has every fourth warp) issues its warps' steps one after the other, or a warp's steps take their
      // latency; before that the tokens' rows are laid out by every block, after it threads add what the warps that split K have,
      // and ranks what the others have.  What it is for: 1 x 4096 x 4096 takes 4.7 us in blocks of two tile warps and 6.1 in
      // clusters of four, gated 8 x 4096 x 2 * 12288 17.1 with sixteen tile warps and 29.7 with sixteen that split K.  The constants are
      // fitted to 7 thousand timings (K 512 to 12288, 64 to 12288 columns, 1 to 32 tokens, all ways to split): the choice is 0.7 %
      // slower than the fastest way on average, 15 % at most; 1.4 % and 22 % at sizes that they were not fitted to.
      int issued = (block_tiles + 3) / 4 * each;
      if (tw < 4) {
        issued = 0;
        for (int k = 0; k < k_warps; k += 4 >> j) issued += each > (k + 1) * steps ? steps : each > k * steps ? each - k * steps : 0;
        issued *= (block_tiles + tw - 1) >> j;
      }
      const double issue = issued * (nt == 1 ? 0.143 : nt == 2 ? 0.2 : nt == 3 ? 0.278 : 0.333);
      const double latency = warp_steps * (0.3 + 0.01 * nt);
      const int rounds = (block_tiles * tokens * cols + kThreads - 1) / kThreads;
      const double sums = ((rounds + ranks - 1) >> i) * ((each + steps - 1) / steps) * 0.063;
      const double cost = waves * (0.7 + (issue > latency ? issue : latency) + each * tokens * 0.0034 + sums) + (ranks > 1 ? 1.5 + 0.07 * i : 0.0);
      if (grid_x == 0 || cost < best) {
        best = cost;
        grid_x = gx;
        p.ranks = ranks; p.units_each = each; p.tile_warps = tw; p.steps = steps;
      }
    }
  }
  I4TC_REQUIRE(grid_x > 0 && chunks <= 65535, I4TC_EUNSUPPORTED, "K is too large, or there are too many tokens for it");
  const size_t smem = w4a16_smem(tokens, small, p.units_each, (p.tiles + grid_x - 1) / grid_x, kWarps / p.tile_warps);
  const dim3 grid((unsigned)grid_x, (unsigned)p.ranks, (unsigned)chunks);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto pick = [&](auto type) {
    using T = decltype(type);
    return gated ? (per_channel ? launch_tokens<T, true, true>(p, grid, smem, st) : launch_tokens<T, true, false>(p, grid, smem, st))
                 : (per_channel ? launch_tokens<T, false, true>(p, grid, smem, st) : launch_tokens<T, false, false>(p, grid, smem, st));
  };
  return dtype == I4TC_BF16 ? pick(__nv_bfloat16{}) : pick(__half{});
}
