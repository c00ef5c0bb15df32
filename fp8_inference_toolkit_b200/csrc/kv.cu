// A paged cache of keys and values: rows appended to it, and attention of a few new tokens over it.
//
// Cache: keys and values [pages, page_size, kv_heads, D] each (any strides with contiguous heads' elements); a sequence's token
// j lies in page block_table[b, j / page_size], row j % page_size.
#include "common.cuh"
#include "ptx.cuh"
#include <float.h>
#include <math.h>
#include <math_constants.h>
#include <type_traits>

namespace i4tc {

namespace {

constexpr unsigned kStatusRange = 4u;   // status word: a block table entry, a length or an index out of range

// ---- append ------------------------------------------------------------------------------------------------------------
// Row i < counts[b] of sequence b, taken from new row select[b, i] (i without select), goes to token lengths[b] + i.  Bound: the rows
// read and written once.  A block takes a few rows; their places are looked up once, by a thread each.  A prompt of 8000 tokens of 8
// heads of 128: 13.7 us with four accesses of a thread on their way together, 15.5 one by one.
constexpr int kAppendThreads = 256, kAppendAtOnce = 4;   // AtOnce: a thread's accesses on their way together

struct AppendParams {
  const void *k, *v;
  void *k_cache, *v_cache;
  long long new_batch, new_token, new_head, page_stride, slot_stride, head_stride;   // bytes
  const int *table, *lengths, *counts, *select;
  long long table_stride, select_stride;
  int batch, tokens, heads, row_units;   // row_units: accesses of one head
  int pages, page_size, table_width;
  int rows_each;                         // of a block
  unsigned int* status;
};

template <typename V>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const AppendParams p) {
  __shared__ long long from[kAppendThreads], to[kAppendThreads];
  pdl_wait();
  const long long row0 = (long long)blockIdx.x * p.rows_each, rows = (long long)p.batch * p.tokens;
  const int n = (int)min((long long)p.rows_each, rows - row0);
  if (threadIdx.x < n) {
    const long long row = row0 + threadIdx.x;
    const int b = (int)(row / p.tokens), i = (int)(row - (long long)b * p.tokens);
    const int count = p.counts ? p.counts[b] : p.tokens;
    long long src = -1, dst = -1;
    bool bad = count < 0 || count > p.tokens;
    if (i < count && !bad) {
      const int pick = p.select ? p.select[b * p.select_stride + i] : i;
      const long long at = (long long)p.lengths[b] + i;
      bad = pick < 0 || pick >= p.tokens || at < i || at >= (long long)p.table_width * p.page_size;
      if (!bad) {
        const int slot = (int)(at % p.page_size), page = p.table[b * p.table_stride + at / p.page_size];
        bad = page < 0 || page >= p.pages;
        if (!bad) {
          src = b * p.new_batch + pick * p.new_token;
          dst = page * p.page_stride + slot * p.slot_stride;
        }
      }
    }
    if (bad) atomicOr(p.status, kStatusRange);
    from[threadIdx.x] = src;
    to[threadIdx.x] = dst;
  }
  __syncthreads();
  const int per_row = 2 * p.heads * p.row_units;   // keys, then values
  for (int i0 = threadIdx.x; i0 < n * per_row; i0 += kAppendThreads * kAppendAtOnce) {
    V held[kAppendAtOnce];
    char* dst[kAppendAtOnce];
#pragma unroll
    for (int k = 0; k < kAppendAtOnce; ++k) {
      const int i = i0 + k * kAppendThreads;
      dst[k] = nullptr;
      if (i < n * per_row) {
        const int r = i / per_row, j = i - r * per_row;
        const bool value = j >= per_row / 2;
        const int c = value ? j - per_row / 2 : j, head = c / p.row_units, unit = c - head * p.row_units;
        if (to[r] >= 0) {
          held[k] = reinterpret_cast<const V*>(static_cast<const char*>(value ? p.v : p.k) + from[r] + head * p.new_head)[unit];
          dst[k] = static_cast<char*>(value ? p.v_cache : p.k_cache) + to[r] + head * p.head_stride + unit * sizeof(V);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAppendAtOnce; ++k)
      if (dst[k] != nullptr) *reinterpret_cast<V*>(dst[k]) = held[k];
  }
}

// ---- attention ---------------------------------------------------------------------------------------------------------
//   out[b, t, h] = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale * q[b, t, h] . k_j)
// over the lengths[b] cached tokens of the sequence and those new tokens j that mask[b, t, j] names (the first t + 1 without a mask);
// nothing visible gives zeros.  Query heads h of one group (heads / kv_heads) read the same keys and values.
//
// Bound: keys and values of the cache, read once: the T new tokens of the heads of a group are the rows of one tile, so a
// key's 2 D bytes serve T * group rows (64 at sixteen drafts of four heads: 64 operations a byte, below what mma.sync gives; a
// tcgen05 tile of 128 rows would be padding for nearly all trees).  One pass with the running maximum and sum of the softmax.
//
// The work is 64-key tiles.  The tiles of all sequences stand in one line, which is cut into equal parts, and every (kv head, row tile) has
// a block for each part: ragged lengths, one long sequence and many short ones all keep every block busy alike, and the heads of
// a token, side by side in a page, are read at the same time.  A part begins and ends anywhere; what it holds of a sequence goes out
// as the result where it holds all of it, else as maximum, sum and weighted values (fp32) to scratch, and a second kernel adds a
// sequence's parts in ascending order.  No atomics: the same bits in every run.
//
// Short sequences (by the room in their table) take another way, without scratch and in one kernel: a cluster of up to eight blocks
// shares one (sequence, kv head, row tile), each takes an equal run of its tiles, and the blocks' sums are added in order through
// distributed shared memory.  One token over 1001 takes 9.4 us on the device, and the host one
// launch and one allocation less (13 us a call instead of 19).
//
// Scores, maxima, sums and values are fp32; a weight is rounded to the values' type (at most 2^-8 of it, fp16 2^-11) before it multiplies them, as
// the tensor instruction takes both operands in one type, and carrying its remainder would double those instructions.  The sum runs
// over the weights as they were rounded, so that an error only shifts the average: off from 64 bits by 2.1e-3 to 2.3e-3 of the
// 2-norm (bf16), 1.7e-3 of it the result's own rounding.
//
// A block's four warps are WR row warps (16 rows each) times 4 / WR key warps, which share out a tile's keys and are added at the
// item's end: few rows do not leave warps idle.  Tiles arrive by cp.async, two ahead; a key's address (its page) is looked
// up one tile before that.
//
// Measured (device time, 32 heads, 8 key heads of 128, bf16): a tree of 16 over 32765 tokens 45.0 us (134 MB), 32 trees of 8 over up to
// 8191 124 us (609 MB, 4.9 TB/s), one token a sequence there 112 us; from 32768 to 65536 tokens of one sequence 20 us more with one
// token (the copy rate) and 30 with sixteen (ldmatrix and mma.sync of 64 rows).
constexpr int kTile = 64, kStages = 3, kAttendThreads = 128, kPlaces = 4, kJoinThreads = 128;

struct AttendParams {
  const void *q, *k, *v, *k_cache, *v_cache;
  const int *table, *lengths;
  const uint8_t* mask;
  void* out;
  float* scratch;
  long long q_batch, q_token, q_head, new_batch, new_token, new_head, page_stride, slot_stride, head_stride;   // elements
  long long table_stride, mask_batch;
  int batch, tokens, heads, kv_heads, group, D;
  int pages, page_size, table_width;
  int rows, row_tiles;          // of an item: tokens * group
  int lines;                    // kv heads times row tiles: blocks of a part
  int parts;                    // of the line, at most
  int ranks;                    // blocks of a cluster, where a sequence has its own; else 0
  float scale_log2;             // |scale| * log2(e), not zero: what is masked stays so
  int negative;                 // the scale's sign
  unsigned int* status;
};

__device__ __forceinline__ int cached(const AttendParams& p, int b, bool report) {
  const int n = p.lengths[b];
  const int most = p.table_width * p.page_size;
  if (n >= 0 && n <= most) return n;
  if (report) atomicOr(p.status, kStatusRange);
  return n < 0 ? 0 : most;
}
__device__ __forceinline__ int tiles_of(const AttendParams& p, int length) { return (length + p.tokens + kTile - 1) / kTile; }

// The line, as a whole warp sees it: its length, and where sequences stand in it.  With up to 32
// sequences a lane keeps its own, so that lengths are read once.
struct Line {
  int length, mine, incl, total;   // of the first 32 sequences: this lane's length and tiles, and the tiles up to it
  __device__ __forceinline__ void open(const AttendParams& p, bool report) {
    const int lane = threadIdx.x & 31;
    length = lane < p.batch ? cached(p, lane, report) : 0;
    mine = lane < p.batch ? tiles_of(p, length) : 0;
    incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    total = __shfl_sync(0xffffffffu, incl, 31);
    if (p.batch > 32) {
      int more = 0;
      for (int b = 32 + lane; b < p.batch; b += 32) more += tiles_of(p, cached(p, b, report));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
      total += more;
    }
  }
  __device__ __forceinline__ int length_of(const AttendParams& p, int b) const {
    return b < 32 ? __shfl_sync(0xffffffffu, length, b) : b < p.batch ? cached(p, b, false) : 0;
  }
  // Tiles before sequence `upto`.
  __device__ __forceinline__ int before(const AttendParams& p, int upto) const {
    if (upto < 32) return __shfl_sync(0xffffffffu, incl - mine, upto);
    int more = 0;
    for (int b = 32 + (threadIdx.x & 31); b < upto; b += 32) more += tiles_of(p, cached(p, b, false));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) more += __shfl_xor_sync(0xffffffffu, more, o);
    return more + __shfl_sync(0xffffffffu, incl, 31);
  }
  // The sequence that holds tile `at`, and the tiles before it.
  __device__ __forceinline__ int find(const AttendParams& p, int at, int& start) const {
    int b0 = 0, base = 0, m = mine, upto = incl;
    for (;;) {
      const unsigned past = __ballot_sync(0xffffffffu, base + upto > at);
      if (past || b0 + 32 >= p.batch) {
        const int l = past ? __ffs(past) - 1 : 31;
        start = base + __shfl_sync(0xffffffffu, upto - m, l);
        return b0 + l;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
      b0 += 32;
      const int lane = threadIdx.x & 31;
      m = b0 + lane < p.batch ? tiles_of(p, cached(p, b0 + lane, false)) : 0;
      upto = m;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
      }
    }
  }
};
// Part i of the line begins at floor(i total / parts); the part that holds tile `at` is the last whose start is not behind it.
__device__ __forceinline__ int part_start(int total, int parts, int part) { return total / parts * part + total % parts * part / parts; }
__device__ __forceinline__ int part_of(int total, int parts, int at) { return (int)(((unsigned long long)(at + 1u) * parts - 1u) / (unsigned)total); }

// Walks the line tile by tile.
struct Cursor {
  int b, tile, tiles, length;
  __device__ __forceinline__ void open(const AttendParams& p, const Line& line) {
    length = line.length_of(p, b);
    tiles = tiles_of(p, length);
  }
  template <bool OWN>
  __device__ __forceinline__ void next(const AttendParams& p, const Line& line) {
    if (++tile < tiles || OWN) return;
    tile = 0;
    ++b;
    open(p, line);
  }
};

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
template <bool TRANS>
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  if constexpr (TRANS)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, uint32_t bytes) {   // 16 bytes, or with 0 zeros: nothing is read then
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2 ulp, far below the rounding of a weight
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Whether any of the new tokens is visible to token t of sequence b.
__device__ __forceinline__ bool sees_new(const AttendParams& p, int b, int t) {
  if (p.mask == nullptr) return true;
  const uint8_t* m = p.mask + b * p.mask_batch + (long long)t * p.tokens;
  for (int j = 0; j < p.tokens; ++j)
    if (m[j]) return true;
  return false;
}
// 1 / sum of a row.  A sum of zero is a row that sees nothing (zeros) or one whose every score is -inf (not a number, as the formula gives).
__device__ __forceinline__ float inverse_sum(const AttendParams& p, float sum, int b, int t, int length) {
  if (sum != 0.f) return 1.0f / sum;
  return length > 0 || sees_new(p, b, t) ? CUDART_NAN_F : 0.f;
}

// Scratch of a part: two slots (the item it begins in, the item it ends in) of maximum [rows], sum [rows], values [rows][DP].
__host__ __device__ constexpr size_t slot_floats(int rows, int dp) { return (size_t)rows * (dp + 2); }

template <int DP, int WR>
struct AttendShape {
  static constexpr int ROWS = 16 * WR, WK = 4 / WR, KEYS = kTile / WK;   // KEYS: of a tile, a warp's share
  static constexpr int kStage = kTile * DP * 2;                          // bytes of a tile's keys, and of its values
  static constexpr int kMerge = WK > 1 ? ROWS * (DP / 2 + 2) * 4 : 0;   // half of the elements of one key warp's rows
  static constexpr int kSmem = kStages * 2 * kStage + kPlaces * kTile * 16 + kMerge;
};

// DP: D rounded up to 64 or 128 (the elements behind D are zeros in shared memory).  OWN: a cluster for each sequence and line.
template <typename T, int DP, int WR, bool OWN>
__global__ void __launch_bounds__(kAttendThreads) attend_kernel(const AttendParams p) {
  using S = AttendShape<DP, WR>;
  constexpr int CH = DP / 8;                        // 16-byte chunks of a row
  constexpr int KS = DP / 16, NT = S::KEYS / 8, DT = DP / 8;
  // Weights are 2^kLift exp(score - m), where m is the largest score up to the last time that a larger one was more than 2^kSlack times
  // its weight: results are seldom scaled anew.  A fp16 weight goes up to 2^14 and keeps 24 + 8 bits below m's.
  constexpr uint32_t kOnes = std::is_same_v<T, __half> ? 0x3C003C00u : 0x3F803F80u;
  constexpr float kLift = std::is_same_v<T, __half> ? 8.f : 0.f, kSlack = std::is_same_v<T, __half> ? 6.f : 8.f;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t stage0 = ptx::smem_u32(smem);
  ulonglong2* places = reinterpret_cast<ulonglong2*>(smem + kStages * 2 * S::kStage);     // [kPlaces][kTile] keys, values
  const uint32_t places_at = stage0 + kStages * 2 * S::kStage;
  float* merge = reinterpret_cast<float*>(smem + kStages * 2 * S::kStage + kPlaces * kTile * 16);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp % WR, wk = warp / WR;
  const int g = lane >> 2, t4 = lane & 3;
  pdl_wait();
  pdl_trigger();

  const int block = OWN ? blockIdx.x / p.ranks : blockIdx.x, rank = OWN ? blockIdx.x % p.ranks : 0;
  const int part = block / p.lines, kvh = block % p.lines / p.row_tiles, tile_row0 = block % p.lines % p.row_tiles * S::ROWS;
  Line line;
  Cursor cur;
  int count;
  if constexpr (OWN) {
    cur.b = part;
    cur.length = cached(p, part, rank == 0);
    cur.tiles = tiles_of(p, cur.length);
    cur.tile = part_start(cur.tiles, p.ranks, rank);
    count = part_start(cur.tiles, p.ranks, rank + 1) - cur.tile;
  } else {
    line.open(p, blockIdx.x == 0);
    const int parts = min(p.parts, line.total);     // no part is empty
    if (part >= parts) return;
    const int first = part_start(line.total, parts, part);
    count = part_start(line.total, parts, part + 1) - first;
    int before;
    cur.b = line.find(p, first, before);
    cur.open(p, line);
    cur.tile = first - before;
  }
  Cursor ahead = cur;                               // whose places are looked up next

  uint32_t q[KS][4];
  float o[DT][4], m[2], l[4];                       // m: reference of the weights, not yet scaled; l: sums of the weights (rows g, and 8 + g from l[2])
  int tok[2];                                       // of this lane's two rows; -1 behind the last
  // This lane's rows are the same for every sequence; its queries of sequence b, and a sequence's running state.
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int row = tile_row0 + wr * 16 + g + 8 * h;
    tok[h] = row < p.rows ? row / p.group : -1;
  }
  auto load_queries = [&](int b, uint32_t (&to)[KS][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int row = tile_row0 + wr * 16 + g + 8 * h;
      const T* src = static_cast<const T*>(p.q) + b * p.q_batch + (long long)(row / p.group) * p.q_token +
                     (long long)(kvh * p.group + row % p.group) * p.q_head;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int d = ks * 16 + e * 8 + 2 * t4;
          to[ks][2 * e + h] = tok[h] >= 0 && d < p.D ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
        }
    }
  };
  auto begin = [&]() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      m[h] = -CUDART_INF_F;
      l[2 * h] = l[2 * h + 1] = 0.f;
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int k = 0; k < 4; ++k) o[dt][k] = 0.f;
  };
  // Before the first tiles: behind their copies the queries came 5 us later (all blocks ask for 19 MB then).
  load_queries(cur.b, q);
  begin();

  // Places of the tile at `ahead`: key tid of it.  In two halves, the page's number and the addresses, so that nobody waits for the table.
  // Where there is no place some row that exists: behind the new tokens nobody sees it; for a page out of range its sequence's result means
  // nothing, and the status word says so.
  auto look_up = [&](const Cursor& ahead) -> int {
    const int j = ahead.tile * kTile + tid;
    return j < ahead.length ? __ldg(p.table + ahead.b * p.table_stride + j / p.page_size) : 0;
  };
  auto place_of = [&](const Cursor& ahead, int page) -> ulonglong2 {
    const int j = ahead.tile * kTile + tid;
    const char *k = static_cast<const char*>(p.k), *v = static_cast<const char*>(p.v);
    long long at = ahead.b * p.new_batch + min(max(j - ahead.length, 0), p.tokens - 1) * p.new_token + kvh * p.new_head;
    if (j < ahead.length) {
      if (page >= 0 && page < p.pages) {
        at = page * p.page_stride + (j % p.page_size) * p.slot_stride + kvh * p.head_stride;
        k = static_cast<const char*>(p.k_cache);
        v = static_cast<const char*>(p.v_cache);
      } else {
        atomicOr(p.status, kStatusRange);
      }
    }
    return make_ulonglong2(reinterpret_cast<unsigned long long>(k + at * 2), reinterpret_cast<unsigned long long>(v + at * 2));
  };
  // Tile i of the part into its stage; the first `rows` of its keys exist, the others become zeros.
  const int my_chunk = tid % CH, my_row = tid / CH;
  const uint32_t in_head = my_chunk * 8 < p.D ? 16u : 0u;
  auto issue = [&](int i, int rows) {
    const uint32_t place = places_at + ((i % kPlaces) * kTile + my_row) * 16;
    const uint32_t dk = stage0 + (i % kStages) * 2 * S::kStage + my_row * (DP * 2) + ((my_chunk ^ (my_row & 7)) * 16);
    constexpr int STEP = kAttendThreads / CH;       // rows apart; a multiple of eight, so that the swizzle stays
    static_assert(STEP % 8 == 0, "rows of a thread share their swizzle");
#pragma unroll
    for (int r = 0; r < kTile; r += STEP) {
      const uint4 at = ptx::lds128(place + r * 16);
      const char* pk = reinterpret_cast<const char*>(at.x | (unsigned long long)at.y << 32) + my_chunk * 16;
      const char* pv = reinterpret_cast<const char*>(at.z | (unsigned long long)at.w << 32) + my_chunk * 16;
      const uint32_t n = r + my_row < rows ? in_head : 0u;
      cp_async_16(dk + r * (DP * 2), pk, n);
      cp_async_16(dk + S::kStage + r * (DP * 2), pv, n);
    }
  };
  int rows[kStages], pages[kStages];                // of the tiles ahead: keys that exist, and this thread's page
  Cursor at[kStages];
#pragma unroll
  for (int i = 0; i < kStages; ++i) {
    at[i] = ahead;
    rows[i] = ahead.length + p.tokens - ahead.tile * kTile;
    pages[i] = 0;
    if (i < count) {
      if (tid < kTile) pages[i] = look_up(ahead);
      ahead.next<OWN>(p, line);
    }
  }
#pragma unroll
  for (int i = 0; i < kStages; ++i)
    if (i < count && tid < kTile) places[i * kTile + tid] = place_of(at[i], pages[i]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < count) issue(i, rows[i]);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  int next_rows = rows[kStages - 1];                // of the tile to be issued next

  // Where this lane reads a tile's keys and values for ldmatrix: chunk c of a row stands at c ^ (row & 7), so chunks 2 j + {0, 1} of eight
  // are four addresses, and the rest (other rows, the next eight chunks) is added to them.
  const int key0 = wk * S::KEYS;                    // this warp's keys in a tile
  uint32_t k_at[4], v_at[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int kr = key0 + (lane & 7) + ((lane >> 4) & 1) * 8, vr = key0 + (lane & 15);
    k_at[j] = stage0 + kr * (DP * 2) + (((2 * j + ((lane >> 3) & 1)) ^ (kr & 7)) * 16);
    v_at[j] = stage0 + S::kStage + vr * (DP * 2) + (((2 * j + (lane >> 4)) ^ (vr & 7)) * 16);
  }
  bool whole = cur.tile == 0;                       // this part has the item from its start

  int stage = 0;                                    // of tile i
  uint32_t next_q[KS][4] = {};
  bool asked = false;
  for (int i = 0; i < count; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
    __syncthreads();
    if (i + kStages - 1 < count) issue(i + kStages - 1, next_rows);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const bool more = i + kStages < count;
    int page = 0;
    if (more && tid < kTile) page = look_up(ahead);
    next_rows = ahead.length + p.tokens - ahead.tile * kTile;
    // the next sequence's queries, two tiles before they are wanted: among the copies they take microseconds
    if (!OWN && !asked && cur.tile + 3 >= cur.tiles && i + cur.tiles - cur.tile < count) {
      load_queries(cur.b + 1, next_q);
      asked = true;
    }

    const uint32_t at_stage = stage * 2 * S::kStage, sv = stage0 + at_stage + S::kStage;
    if (++stage == kStages) stage = 0;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) s[nt][k] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int np = 0; np < NT / 2; ++np) {
        uint32_t b[4];
        ldmatrix4<false>(b, k_at[ks & 3] + at_stage + (np * 16 * (DP * 2) + (ks >> 2) * 128));
        mma<T>(s[2 * np], q[ks], b[0], b[1]);
        mma<T>(s[2 * np + 1], q[ks], b[2], b[3]);
      }
    if (p.negative) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) s[nt][k] = -s[nt][k];
    }
    const int j0 = cur.tile * kTile;
    const bool edge = j0 + kTile > cur.length;      // the tile holds new tokens, or what is behind them
    bool odd = false;
    if (edge) {
      // Which of this lane's keys its two rows see, as bits: the cached ones, then the row's bits of the mask (four lanes have a row and
      // read a quarter of them each).  Rolled, as is the next loop: an item comes here once, and what it does not run it need not fetch.
      const int rel = cur.length - (j0 + key0 + 2 * t4);
      uint64_t seen[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint64_t bits = 0;
        if (tok[h] >= 0) {
          if (p.mask == nullptr) {
            bits = ~0ull >> (63 - tok[h]);
          } else {
            const uint8_t* row = p.mask + cur.b * p.mask_batch + (long long)tok[h] * p.tokens;
#pragma unroll 2
            for (int j = t4; j < p.tokens; j += 4) bits |= (uint64_t)(row[j] != 0) << j;
          }
        }
        bits |= __shfl_xor_sync(0xffffffffu, bits, 1);
        bits |= __shfl_xor_sync(0xffffffffu, bits, 2);
        seen[h] = rel >= 64 ? ~0ull : rel > 0 ? bits << rel | ((1ull << rel) - 1) : rel > -64 ? bits >> -rel : 0ull;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (!(seen[k >> 1] >> (nt * 8 + (k & 1)) & 1)) s[nt][k] = -CUDART_INF_F;
      // Not only the scores of what a row does not see: its values may be infinite or no numbers, which a weight of zero does not undo.
#pragma unroll 1
      for (int r = tid; r < kTile * CH; r += kAttendThreads) {
        const int key = r / CH, c = r % CH;
        if (j0 + key < cur.length) continue;
        const uint32_t at = sv + key * (DP * 2) + ((c ^ (key & 7)) * 16);
        constexpr uint32_t kExp = std::is_same_v<T, __half> ? 0x7C007C00u : 0x7F807F80u;
        uint4 v = ptx::lds128(at);
        const uint32_t x = __vcmpeq2(v.x & kExp, kExp), y = __vcmpeq2(v.y & kExp, kExp), z = __vcmpeq2(v.z & kExp, kExp), w = __vcmpeq2(v.w & kExp, kExp);
        if (x | y | z | w) {
          ptx::sts128(at, make_uint4(v.x & ~x, v.y & ~y, v.z & ~z, v.w & ~w));
          odd = true;
        }
      }
      odd = __syncthreads_or(odd);
    }

    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 4; ++k) top[k >> 1] = fmaxf(top[k >> 1], s[nt][k]);
    float base[2];
    bool rise = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
      rise |= m[h] == -CUDART_INF_F ? top[h] != m[h] : (top[h] - m[h]) * p.scale_log2 > kSlack;
    }
    if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float fade = m[h] == top[h] ? 1.f : exp2_fast((m[h] - top[h]) * p.scale_log2);
        m[h] = top[h];
        l[2 * h] *= fade;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          o[dt][2 * h] *= fade;
          o[dt][2 * h + 1] *= fade;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) base[h] = m[h] == -CUDART_INF_F ? 0.f : m[h] * p.scale_log2 - kLift;
    if (odd) {                                      // what was taken out of the values goes to the rows that see it
#pragma unroll 1
      for (int key = key0; key < key0 + S::KEYS; ++key) {
        const int j = j0 + key - cur.length;
        if (j < 0 || j >= p.tokens) continue;
        const T* src = static_cast<const T*>(p.v) + cur.b * p.new_batch + j * p.new_token + kvh * p.new_head;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = tok[h];
          if (t < 0 || !(p.mask ? p.mask[cur.b * p.mask_batch + (long long)t * p.tokens + j] != 0 : j <= t)) continue;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const int d = dt * 8 + 2 * t4;
            if (d < p.D) {
              const float x = to_f32(src[d]), y = to_f32(src[d + 1]);
              if (!isfinite(x)) o[dt][2 * h] += x;
              if (!isfinite(y)) o[dt][2 * h + 1] += y;
            }
          }
        }
      }
    }
    uint32_t w[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        w[nt][h] = pack_pair<T>(exp2_fast(fmaf(s[nt][2 * h], p.scale_log2, -base[h])), exp2_fast(fmaf(s[nt][2 * h + 1], p.scale_log2, -base[h])));
#pragma unroll
    for (int kk = 0; kk < NT / 2; ++kk) {
      const uint32_t a[4] = {w[2 * kk][0], w[2 * kk][1], w[2 * kk + 1][0], w[2 * kk + 1][1]};
      mma<T>(l, a, kOnes, kOnes);                   // the sums of the weights as they were rounded
#pragma unroll
      for (int dp = 0; dp < DT / 2; ++dp) {
        uint32_t b[4];
        ldmatrix4<true>(b, v_at[dp & 3] + at_stage + (kk * 16 * (DP * 2) + (dp >> 2) * 128));
        mma<T>(o[2 * dp], a, b[0], b[1]);
        mma<T>(o[2 * dp + 1], a, b[2], b[3]);
      }
    }

    const bool ends = cur.tile + 1 == cur.tiles;
    if (ends || i + 1 == count) {
      m[0] *= p.scale_log2;
      m[1] *= p.scale_log2;
      if constexpr (S::WK > 1) {
        // the key warps, one after the other and half of the elements at a time, into the first
        float* mo = merge + (wr * 16 + g) * (DP / 2) + 2 * t4;
        float* ml = merge + S::ROWS * (DP / 2) + (wr * 16 + g) * 2;
#pragma unroll 1
        for (int from = 1; from < S::WK; ++from) {
          float fa[2], fb[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            __syncthreads();
            if (wk == from) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int dt = 0; dt < DT / 2; ++dt)
                  *reinterpret_cast<float2*>(mo + 8 * h * (DP / 2) + dt * 8) =
                      make_float2(o[half * (DT / 2) + dt][2 * h], o[half * (DT / 2) + dt][2 * h + 1]);
                if (half == 0 && t4 == 0) *reinterpret_cast<float2*>(ml + 16 * h) = make_float2(m[h], l[2 * h]);
              }
            }
            __syncthreads();
            if (wk == 0) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (half == 0) {
                  const float2 his = *reinterpret_cast<const float2*>(ml + 16 * h);
                  const float both = fmaxf(m[h], his.x), zero = both == -CUDART_INF_F ? 0.f : both;
                  fa[h] = exp2_fast(m[h] - zero);
                  fb[h] = exp2_fast(his.x - zero);
                  m[h] = both;
                  l[2 * h] = l[2 * h] * fa[h] + his.y * fb[h];
                }
#pragma unroll
                for (int dt = 0; dt < DT / 2; ++dt) {
                  const float2 v = *reinterpret_cast<const float2*>(mo + 8 * h * (DP / 2) + dt * 8);
                  float* mine = o[half * (DT / 2) + dt] + 2 * h;
                  mine[0] = mine[0] * fa[h] + v.x * fb[h];
                  mine[1] = mine[1] * fa[h] + v.y * fb[h];
                }
              }
            }
          }
        }
      }
      if (wk == 0) {
        const int row0 = tile_row0 + wr * 16 + g;
        if (OWN && p.ranks > 1) {
          // added below
        } else if (OWN || (whole && ends)) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = row0 + 8 * h;
            if (tok[h] < 0) continue;
            const float inv = inverse_sum(p, l[2 * h], cur.b, tok[h], cur.length);
            T* dst = static_cast<T*>(p.out) + (((long long)cur.b * p.tokens + tok[h]) * p.heads + kvh * p.group + row % p.group) * p.D;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
              const int d = dt * 8 + 2 * t4;
              if (d < p.D) *reinterpret_cast<uint32_t*>(dst + d) = pack_pair<T>(o[dt][2 * h] * inv, o[dt][2 * h + 1] * inv);
            }
          }
        } else {
          // the item the part began in, or (where that is another) the one it ends in
          const bool opening = !whole || i == cur.tile;
          float* slot = p.scratch + ((size_t)blockIdx.x * 2 + (opening ? 0 : 1)) * slot_floats(S::ROWS, DP);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int row = wr * 16 + g + 8 * h;
            if (t4 == 0) {
              slot[row] = m[h];
              slot[S::ROWS + row] = l[2 * h];
            }
            float* dst = slot + 2 * S::ROWS + row * DP + 2 * t4;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float2*>(dst + dt * 8) = make_float2(o[dt][2 * h], o[dt][2 * h + 1]);
          }
        }
      }
      whole = true;
    }
    const bool another = !OWN && ends && i + 1 < count;
    cur.next<OWN>(p, line);
    if (another) {
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int k = 0; k < 4; ++k) q[ks][k] = next_q[ks][k];
      begin();
      asked = false;
    }
    if (more) {
      if (tid < kTile) places[((i + kStages) % kPlaces) * kTile + tid] = place_of(ahead, page);
      ahead.next<OWN>(p, line);
    }
  }
  if constexpr (OWN) {
    if (p.ranks == 1) return;
    // this block's sums where its tiles were, then every rank adds the rows rank, rank + ranks, ...
    float* sums = reinterpret_cast<float*>(smem);   // values [rows][DP], then reference and sum [rows][2]
    static_assert(S::ROWS * (DP + 2) * 4 <= kStages * 2 * S::kStage, "the sums fit the tiles' place");
    __syncthreads();
    if (wk == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = wr * 16 + g + 8 * h;
        float* dst = sums + row * DP + 2 * t4;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float2*>(dst + dt * 8) = make_float2(o[dt][2 * h], o[dt][2 * h + 1]);
        if (t4 == 0) *reinterpret_cast<float2*>(sums + S::ROWS * DP + row * 2) = make_float2(m[h], l[2 * h]);
      }
    }
    ptx::cluster_sync();
    constexpr int E = DP / 32;
    const uint32_t base = stage0;
    for (int row = rank + p.ranks * warp; row < S::ROWS && tile_row0 + row < p.rows; row += p.ranks * (kAttendThreads / 32)) {
      float top = -CUDART_INF_F, sum = 0.f, v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.f;
      float ms[8], ls[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ms[k] = -CUDART_INF_F;
        ls[k] = 0.f;
        if (k < p.ranks)
          asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(ms[k]), "=f"(ls[k]) : "r"(ptx::mapa_shared(base + (S::ROWS * DP + row * 2) * 4, k)));
        top = fmaxf(top, ms[k]);
      }
      const float zero = top == -CUDART_INF_F ? 0.f : top;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k >= p.ranks) break;
        const float f = exp2_fast(ms[k] - zero);
        sum += ls[k] * f;
        const uint32_t from = ptx::mapa_shared(base + (row * DP + lane * E) * 4, k);
        float x[E];
        if constexpr (E == 4) asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]) : "r"(from));
        else asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(x[0]), "=f"(x[1]) : "r"(from));
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += x[e] * f;
      }
      const int r = tile_row0 + row, t = r / p.group;
      const float inv = inverse_sum(p, sum, part, t, cached(p, part, false));
      T* dst = static_cast<T*>(p.out) + (((long long)part * p.tokens + t) * p.heads + kvh * p.group + r % p.group) * p.D + lane * E;
#pragma unroll
      for (int e = 0; e < E; e += 2)
        if (lane * E + e < p.D) *reinterpret_cast<uint32_t*>(dst + e) = pack_pair<T>(v[e] * inv, v[e + 1] * inv);
    }
    ptx::cluster_sync();   // the others may still be reading
  }
}

// Sequences that no part held whole: their parts in ascending order.  A block takes rows_each rows of a (sequence, line).  Few parts: a warp
// has a row to itself.  More: the block's warps take a quarter of the parts each, and these are added in order.  A lane has DP / 32
// consecutive elements.
template <typename T, int DP>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(const AttendParams p, int tile_rows, int rows_each) {
  constexpr int E = DP / 32, WARPS = kJoinThreads / 32, AT_ONCE = 8;   // AT_ONCE: parts whose loads are on their way together
  __shared__ float sums[WARPS][DP + 2];
  // The lengths may be read before the wait: the kernel before this one let it start after its own wait, and writes scratch and results only.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.x / p.lines, at_line = blockIdx.x % p.lines, row0 = blockIdx.y * rows_each;
  Line line;
  line.open(p, false);
  const int length = line.length_of(p, b), tiles = tiles_of(p, length);
  const int start = line.before(p, b);
  const int parts = min(p.parts, line.total);
  const int first = part_of(line.total, parts, start), last = part_of(line.total, parts, start + tiles - 1);
  const size_t slots = 2 * slot_floats(tile_rows, DP), step = slots * p.lines;   // a block's, and from a part to the next
  const bool begins = part_start(line.total, parts, first) == start;
  pdl_wait();
  const int rows = min(rows_each, min(tile_rows, p.rows - at_line % p.row_tiles * tile_rows) - row0);
  if (rows <= 0 || first == last) return;
  const float* scratch = p.scratch;
  pdl_fresh(scratch);
  scratch += at_line * slots;
  const float* opening = scratch + first * step + (begins ? 0 : slots / 2);
  auto slot = [&](int part) { return part == first ? opening : scratch + part * step; };
  float top, sum, v[E];
  auto gather = [&](int row, int from, int to) {    // parts [from, to) of a row into top, sum and v
    top = -CUDART_INF_F;
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
    for (int part = from; part < to; part += AT_ONCE) {
      float m[AT_ONCE], l[AT_ONCE], x[AT_ONCE][E];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        m[k] = -CUDART_INF_F;
        l[k] = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[k][e] = 0.f;
        if (part + k < to) {
          const float* s = slot(part + k);
          m[k] = s[row];
          l[k] = s[tile_rows + row];
          const float* o = s + 2 * tile_rows + row * DP + lane * E;
          if constexpr (E == 4) {
            const float4 q = *reinterpret_cast<const float4*>(o);
            x[k][0] = q.x; x[k][1] = q.y; x[k][2] = q.z; x[k][3] = q.w;
          } else {
            const float2 q = *reinterpret_cast<const float2*>(o);
            x[k][0] = q.x; x[k][1] = q.y;
          }
        }
      }
      float both = top;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) both = fmaxf(both, m[k]);
      const float zero = both == -CUDART_INF_F ? 0.f : both, fade = exp2_fast(top - zero);
      top = both;
      sum *= fade;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] *= fade;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const float f = exp2_fast(m[k] - zero);
        sum += l[k] * f;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += x[k][e] * f;
      }
    }
  };
  auto place = [&](int row, int& t) -> T* {         // of a row's result
    const int r = at_line % p.row_tiles * tile_rows + row, head = at_line / p.row_tiles * p.group + r % p.group;
    t = r / p.group;
    return static_cast<T*>(p.out) + (((long long)b * p.tokens + t) * p.heads + head) * p.D;
  };
  const int count = last - first + 1;
  int t;
  if (count <= AT_ONCE) {
    for (int r = warp; r < rows; r += WARPS) {
      gather(row0 + r, first, last + 1);
      T* dst = place(row0 + r, t) + lane * E;
      const float inv = inverse_sum(p, sum, b, t, length);
#pragma unroll
      for (int e = 0; e < E; e += 2)
        if (lane * E + e < p.D) *reinterpret_cast<uint32_t*>(dst + e) = pack_pair<T>(v[e] * inv, v[e + 1] * inv);
    }
    return;
  }
  const int each = (count + WARPS - 1) / WARPS;
  for (int r = 0; r < rows; ++r) {
    gather(row0 + r, first + min(count, warp * each), first + min(count, (warp + 1) * each));
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) sums[warp][lane * E + e] = v[e];
    if (lane == 0) {
      sums[warp][DP] = top;
      sums[warp][DP + 1] = sum;
    }
    __syncthreads();
    float all = -CUDART_INF_F;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) all = fmaxf(all, sums[k][DP]);
    const float base = all == -CUDART_INF_F ? 0.f : all;
    const int d = threadIdx.x;
    float x = 0.f;
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const float f = exp2_fast(sums[k][DP] - base);
      sum += sums[k][DP + 1] * f;
      if (d < DP) x += sums[k][d] * f;
    }
    T* dst = place(row0 + r, t);
    if (d < p.D) {
      const float y = x * inverse_sum(p, sum, b, t, length);
      if constexpr (std::is_same_v<T, __half>) dst[d] = __float2half_rn(y); else dst[d] = __float2bfloat16_rn(y);
    }
  }
}

int row_warps(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : 4; }
int padded_dim(int64_t D) { return D <= 64 ? 64 : 128; }
// How the work is shared out: clusters of `ranks` blocks for each sequence and line, or (0) parts of the line, two blocks an SM in all.
struct AttendPlan {
  int ranks, parts;
};
AttendPlan attend_plan(int sm_count, int64_t batch, int64_t kv_heads, int64_t rows, int64_t D, int64_t most_length, int64_t tokens) {
  const int warps = row_warps(rows);
  const int64_t row_tiles = (rows + 16 * warps - 1) / (16 * warps), lines = kv_heads * row_tiles;
  const int64_t tiles = (most_length + tokens + kTile - 1) / kTile, slots = (int64_t)sm_count * 2;
  const int64_t most = slots / lines < 1 ? 1 : slots / lines;
  AttendPlan plan = {0, (int)(batch * tiles < most ? batch * tiles : most)};
  // Microseconds, by the room in the table, from 344 sizes timed all five ways (lengths from an eighth of the room to all of it): a block's way
  // to its first tile and its end, its tiles, a cluster's sums; for parts the second kernel (9.4 with everything, and 2.5 of the
  // 5 that a call of it costs the host more).  What it is for, 8 key heads of 128 and 4 query heads each, clusters of 1, 2, 4, 8 | parts: one token
  // over 32000 564 us, 288, 149, 79 | 34; 64 trees of four over up to 256 24, 46, 80, 165 | 33.  The choice is 2.7 % slower on
  // the device than the fastest way on average and 34 % at most; 3.4 % and 46 % at 378 sizes that it was not fitted to.
  const double tile = (warps == 1 ? 1.15 : warps == 2 ? 1.43 : 1.88) * (padded_dim(D) == 64 ? 0.64 : 1.0);
  const int64_t line_rows = rows < 16 * warps ? rows : 16 * warps;
  double best = 9.4 + 2.5 + 0.97 * tile * (double)((batch * tiles + plan.parts - 1) / plan.parts * ((plan.parts * lines + slots - 1) / slots)) +
                0.2e-3 * (double)(batch * lines * line_rows);
  for (int i = 0; i < 4; ++i) {
    const int64_t ranks = 1 << i;
    const double load = (double)(batch * lines * ranks) / ((double)slots * (i < 2 ? 1.0 : i == 2 ? 0.89 : 0.81));   // clusters do not cross a GPC
    const double waves = load <= 1.0 ? 1.0 : 0.87 * load + 0.13 * ceil(load);
    const double cost = 0.4 + waves * (4.6 + tile * (double)((tiles + ranks - 1) / ranks)) + (i > 0 ? 3.5 + 0.36 * i : 0.0);
    if (cost < best && batch * lines * ranks < (1ll << 30)) {
      best = cost;
      plan.ranks = (int)ranks;
    }
  }
  return plan;
}

template <typename T, int DP, int WR, bool OWN>
int launch_attend(const AttendParams& p, cudaStream_t st) {
  using S = AttendShape<DP, WR>;
  auto kernel = attend_kernel<T, DP, WR, OWN>;
  static bool configured[64] = {false};
  int dev = 0;
  I4TC_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !configured[dev]) {
    I4TC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem));
    if (dev < 64) configured[dev] = true;
  }
  if constexpr (OWN) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.batch * p.lines * p.ranks), 1, 1);
    cfg.blockDim = dim3(kAttendThreads, 1, 1);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.ranks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = p.ranks > 1 ? 2 : 1;
    I4TC_CUDA(cudaLaunchKernelEx(&cfg, kernel, p));
  } else {
    I4TC_CUDA(launch_kernel(true, kernel, dim3((unsigned)(p.parts * p.lines)), kAttendThreads, S::kSmem, st, p));
    // A row a block where they are few, more where blocks would queue: 8192 blocks of a row took 14 us longer than 1024 of eight.
    const int rows = S::ROWS < p.rows ? S::ROWS : p.rows, all = p.batch * p.lines * rows;
    const int each = all > 4096 ? 8 : all > 1024 ? 4 : 1;
    const dim3 grid((unsigned)(p.batch * p.lines), (unsigned)((rows + each - 1) / each));
    I4TC_CUDA(launch_kernel(true, attend_join_kernel<T, DP>, grid, kJoinThreads, 0, st, p, S::ROWS, each));
  }
  return I4TC_OK;
}

template <typename T, int DP, bool OWN>
int launch_rows(const AttendParams& p, int warps, cudaStream_t st) {
  return warps == 1 ? launch_attend<T, DP, 1, OWN>(p, st) : warps == 2 ? launch_attend<T, DP, 2, OWN>(p, st) : launch_attend<T, DP, 4, OWN>(p, st);
}
template <typename T>
int launch_dim(const AttendParams& p, int warps, cudaStream_t st) {
  if (padded_dim(p.D) == 64) return p.ranks ? launch_rows<T, 64, true>(p, warps, st) : launch_rows<T, 64, false>(p, warps, st);
  return p.ranks ? launch_rows<T, 128, true>(p, warps, st) : launch_rows<T, 128, false>(p, warps, st);
}

}  // namespace

}  // namespace i4tc

using namespace i4tc;

extern "C" int64_t i4tc_tree_attention_scratch_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t D,
                                                     int64_t most_length, int device) {
  const DeviceInfo* info;
  if (batch <= 0 || tokens <= 0 || heads <= 0 || kv_heads <= 0 || D <= 0 || most_length < 0 || device_info(device, &info) != I4TC_OK) return 0;
  const int64_t rows = tokens * (heads / kv_heads);
  const int tile_rows = 16 * row_warps(rows);
  const int64_t lines = kv_heads * ((rows + tile_rows - 1) / tile_rows);
  const AttendPlan plan = attend_plan(info->sm_count, batch, kv_heads, rows, D, most_length, tokens);
  return plan.ranks ? 0 : plan.parts * lines * 2 * (int64_t)slot_floats(tile_rows, padded_dim(D)) * 4;
}

extern "C" int i4tc_tree_attention(const i4tc_tree_attention_args* a, int device, void* stream) {
  I4TC_REQUIRE(a != nullptr, I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(a->dtype == I4TC_BF16 || a->dtype == I4TC_FP16, I4TC_EUNSUPPORTED, "queries must be bfloat16 or float16");
  I4TC_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->heads >= 0, I4TC_EINVAL, "bad size");
  if (a->batch == 0 || a->tokens == 0 || a->heads == 0) return I4TC_OK;
  I4TC_REQUIRE(a->tokens <= 64, I4TC_EUNSUPPORTED, "at most 64 new tokens a sequence");
  I4TC_REQUIRE(a->head_dim > 0 && a->head_dim <= 128 && a->head_dim % 8 == 0, I4TC_EUNSUPPORTED,
               "heads must have a multiple of 8 and at most 128 elements");
  I4TC_REQUIRE(a->kv_heads > 0 && a->heads % a->kv_heads == 0 && a->heads <= 65536, I4TC_EINVAL, "heads must be a multiple of kv_heads");
  I4TC_REQUIRE(a->batch <= 65536 && a->pages >= 0 && a->pages < (1ll << 31) && a->page_size > 0 && a->page_size < (1ll << 31) &&
                   a->table_width >= 0 && a->table_width < (1ll << 31), I4TC_EINVAL, "bad size");
  I4TC_REQUIRE(isfinite(a->scale) && fabs(a->scale) < 1e30, I4TC_EINVAL, "the scale must be finite");
  I4TC_REQUIRE(a->q && a->k && a->v && a->lengths && a->out, I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(a->table_width == 0 || (a->block_table && (a->pages == 0 || (a->k_cache && a->v_cache))), I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(aligned_to(a->k, 16) && aligned_to(a->v, 16) && aligned_to(a->k_cache, 16) && aligned_to(a->v_cache, 16) &&
                   aligned_to(a->q, 4) && aligned_to(a->out, 16) && aligned_to(a->scratch, 16) && a->q_batch % 2 == 0 && a->q_token % 2 == 0 &&
                   a->q_head % 2 == 0 && (a->new_batch | a->new_token | a->new_head | a->page_stride | a->slot_stride | a->head_stride) % 8 == 0,
               I4TC_EALIGN, "keys and values must be 16-byte aligned, and queries 4-byte");
  const DeviceInfo* info;
  if (int rc = device_info(device, &info)) return rc;
  I4TC_REQUIRE(info->cc_major == 10, I4TC_EDEVICE, "device %d is sm_%d%d; this library needs sm_100", device, info->cc_major, info->cc_minor);
  AttendParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.table = a->block_table; p.lengths = a->lengths; p.mask = a->mask; p.out = a->out; p.scratch = static_cast<float*>(a->scratch);
  p.q_batch = a->q_batch; p.q_token = a->q_token; p.q_head = a->q_head;
  p.new_batch = a->new_batch; p.new_token = a->new_token; p.new_head = a->new_head;
  p.page_stride = a->page_stride; p.slot_stride = a->slot_stride; p.head_stride = a->head_stride;
  p.table_stride = a->table_stride; p.mask_batch = a->mask_batch;
  p.batch = (int)a->batch; p.tokens = (int)a->tokens; p.heads = (int)a->heads; p.kv_heads = (int)a->kv_heads;
  p.group = p.heads / p.kv_heads; p.D = (int)a->head_dim;
  p.pages = (int)a->pages; p.page_size = (int)a->page_size; p.table_width = (int)a->table_width;
  const int64_t rows = (int64_t)p.tokens * p.group;
  const int warps = row_warps(rows);
  p.rows = (int)rows; p.row_tiles = (int)((rows + 16 * warps - 1) / (16 * warps));
  p.lines = p.kv_heads * p.row_tiles;
  const int64_t most_length = a->table_width * a->page_size;
  I4TC_REQUIRE(most_length < (1ll << 31) - 2 * kTile && a->batch * ((most_length + a->tokens) / kTile + 1) < (1ll << 31) && a->batch * p.lines < (1ll << 24),
               I4TC_EUNSUPPORTED, "the table has room for too many tokens");
  const AttendPlan plan = attend_plan(info->sm_count, a->batch, p.kv_heads, rows, p.D, most_length, a->tokens);
  p.parts = plan.parts;
  p.ranks = plan.ranks;
  I4TC_REQUIRE(p.ranks || a->scratch != nullptr, I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(p.ranks || a->scratch_bytes >= (int64_t)p.parts * p.lines * 2 * (int64_t)slot_floats(16 * warps, padded_dim(p.D)) * 4, I4TC_EWORKSPACE,
               "the scratch is too small");
  p.scale_log2 = fmaxf((float)(fabs(a->scale) * 1.4426950408889634), FLT_MIN);
  p.negative = a->scale < 0;
  p.status = info->status;
  DeviceGuard guard(device);
  I4TC_CUDA(guard.err);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return a->dtype == I4TC_BF16 ? launch_dim<__nv_bfloat16>(p, warps, st) : launch_dim<__half>(p, warps, st);
}

extern "C" int i4tc_kv_append(const i4tc_kv_append_args* a, int device, void* stream) {
  I4TC_REQUIRE(a != nullptr, I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(a->element_bytes == 2, I4TC_EUNSUPPORTED, "keys and values must be bfloat16 or float16");
  I4TC_REQUIRE(a->batch >= 0 && a->tokens >= 0 && a->kv_heads >= 0 && a->head_dim >= 0, I4TC_EINVAL, "bad size");
  if (a->batch == 0 || a->tokens == 0 || a->kv_heads == 0 || a->head_dim == 0) return I4TC_OK;
  I4TC_REQUIRE(a->batch < (1ll << 31) && a->tokens < (1ll << 31) && a->kv_heads <= 65536 && a->head_dim <= 2048 && a->pages >= 0 &&
                   a->pages < (1ll << 31) && a->page_size > 0 && a->page_size < (1ll << 31) && a->table_width >= 0 && a->table_width < (1ll << 31),
               I4TC_EINVAL, "bad size");
  I4TC_REQUIRE(a->k && a->v && a->lengths, I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(a->table_width == 0 || (a->block_table && (a->pages == 0 || (a->k_cache && a->v_cache))), I4TC_EINVAL, "null pointer");
  const DeviceInfo* info;
  if (int rc = device_info(device, &info)) return rc;
  AppendParams p = {};
  p.k = a->k; p.v = a->v; p.k_cache = a->k_cache; p.v_cache = a->v_cache;
  p.new_batch = a->new_batch * 2; p.new_token = a->new_token * 2; p.new_head = a->new_head * 2;
  p.page_stride = a->page_stride * 2; p.slot_stride = a->slot_stride * 2; p.head_stride = a->head_stride * 2;
  p.table = a->block_table; p.lengths = a->lengths; p.counts = a->counts; p.select = a->select;
  p.table_stride = a->table_stride; p.select_stride = a->select_stride;
  p.batch = (int)a->batch; p.tokens = (int)a->tokens; p.heads = (int)a->kv_heads;
  p.pages = (int)a->pages; p.page_size = (int)a->page_size; p.table_width = (int)a->table_width;
  p.status = info->status;
  int bytes = 16;   // the widest access that strides, rows and addresses are multiples of
  const long long all = p.new_batch | p.new_token | p.new_head | p.page_stride | p.slot_stride | p.head_stride | a->head_dim * 2;
  while (bytes > 2 && (all % bytes != 0 || !aligned_to(p.k, bytes) || !aligned_to(p.v, bytes) || !aligned_to(p.k_cache, bytes) || !aligned_to(p.v_cache, bytes)))
    bytes /= 2;
  I4TC_REQUIRE(aligned_to(p.k, bytes) && aligned_to(p.v, bytes) && aligned_to(p.k_cache, bytes) && aligned_to(p.v_cache, bytes), I4TC_EALIGN,
               "operands must be aligned to their element size");
  p.row_units = (int)(a->head_dim * 2 / bytes);
  const long long rows = (long long)p.batch * p.tokens, per_row = 2ll * p.heads * p.row_units;
  p.rows_each = (int)(kAppendAtOnce * kAppendThreads / per_row);
  p.rows_each = p.rows_each < 1 || rows <= 2 * info->sm_count ? 1 : p.rows_each > kAppendThreads ? kAppendThreads : p.rows_each;
  const long long blocks = (rows + p.rows_each - 1) / p.rows_each;
  I4TC_REQUIRE(blocks < (1ll << 31) && per_row * p.rows_each < (1ll << 31), I4TC_EINVAL, "bad size");
  DeviceGuard guard(device);
  I4TC_CUDA(guard.err);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto kernel = bytes == 16 ? append_kernel<uint4> : bytes == 8 ? append_kernel<uint2> : bytes == 4 ? append_kernel<uint32_t> : append_kernel<uint16_t>;
  I4TC_CUDA(launch_kernel(true, kernel, dim3((unsigned)blocks), kAppendThreads, 0, st, p));
  return I4TC_OK;
}
