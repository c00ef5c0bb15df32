// Rotary position embedding at given positions.
//
//   (a, b) -> scale * (a cos - b sin, b cos + a sin),  angle = position * f_i  (inverse: minus the angle)
//
// over the first R of D elements of every head; pair i is (i, i + R/2) or (2i, 2i + 1).
//
// Bound: one read and one write of the tensor.  An angle's cosine and sine are computed once per token, for all heads: in turns,
// as a 64-bit product whose whole part is dropped before it becomes a 32-bit argument (positions of a million turn the fastest
// pair 159 thousand times: a 32-bit angle would be off by 0.03 rad, and a bf16 table by 2^-9 at any position).  Both
// halves of the rotation are in one thread, in 16-byte accesses where the operands allow them.  The sums are fp32 and rounded once.
#include "common.cuh"
#include <type_traits>

namespace i4tc {

namespace {

constexpr int kRopeThreads = 256;
constexpr double kTurnsPerRadian = 0.15915494309189533577;   // 1 / (2 pi)

struct RopeParams {
  const void* x;
  void* out;
  long long x_token, x_head, out_token, out_head;   // strides in elements
  const void* positions;                            // int32 or int64
  const double* freqs;                              // [R / 2] radians a position
  int tokens, heads, D, R;
  int heads_each, tokens_each;                      // of a block
  float scale;
  int long_positions, inverse, in_place;
};

template <int BYTES> struct VecOf;
template <> struct VecOf<16> { using type = uint4; };
template <> struct VecOf<8> { using type = uint2; };
template <> struct VecOf<4> { using type = uint32_t; };
template <> struct VecOf<2> { using type = uint16_t; };

template <typename T, int VEC>
struct Chunk {
  using V = typename VecOf<VEC * 2>::type;
  T v[VEC];
  __device__ __forceinline__ void load(const T* p) { *reinterpret_cast<V*>(v) = *reinterpret_cast<const V*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<V*>(p) = *reinterpret_cast<const V*>(v); }
};
__device__ __forceinline__ void put(__nv_bfloat16& d, float v) { d = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half& d, float v) { d = __float2half_rn(v); }

// VEC: elements of one access (with neighbouring pairs and VEC 1 a pair takes two).  INTER: neighbouring elements are a pair, else
// the two halves of the first R.
template <typename T, int VEC, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeParams p) {
  extern __shared__ float2 turn[];                  // [token of the block][R / 2]: cosine and sine, scaled
  pdl_wait();
  const T* x = static_cast<const T*>(p.x);
  const void* positions = p.positions;
  const double* freqs = p.freqs;
  pdl_fresh(x); pdl_fresh(positions); pdl_fresh(freqs);
  const int pairs = p.R / 2, tok0 = blockIdx.x * p.tokens_each, ntok = min(p.tokens_each, p.tokens - tok0);
  const int head0 = blockIdx.y * p.heads_each, nheads = min(p.heads_each, p.heads - head0);
  for (int i = threadIdx.x; i < ntok * pairs; i += kRopeThreads) {
    const int tok = tok0 + i / pairs;
    const double pos = p.long_positions ? (double)static_cast<const long long*>(positions)[tok] : (double)static_cast<const int*>(positions)[tok];
    const double turns = pos * (freqs[i % pairs] * kTurnsPerRadian);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    turn[i] = make_float2(c * p.scale, (p.inverse ? -s : s) * p.scale);
  }
  __syncthreads();
  // a head's accesses: those that turn (one of each half, or neighbours), then, where the result is another tensor, the others
  const int turning = INTER && VEC > 1 ? p.R / VEC : pairs / VEC, each = turning + (p.in_place ? 0 : (p.D - p.R) / VEC);
  const int per_token = nheads * each;
  for (int i = threadIdx.x; i < ntok * per_token; i += kRopeThreads) {
    const int tok = i / per_token, j = i - tok * per_token, head = j / each, c = j - head * each;
    const T* src = x + (long long)(tok0 + tok) * p.x_token + (long long)(head0 + head) * p.x_head;
    T* dst = static_cast<T*>(p.out) + (long long)(tok0 + tok) * p.out_token + (long long)(head0 + head) * p.out_head;
    const float2* cs = turn + tok * pairs;
    if (c >= turning) {
      const int at = p.R + (c - turning) * VEC;
      Chunk<T, VEC> v;
      v.load(src + at);
      v.store(dst + at);
    } else if constexpr (INTER && VEC == 1) {
      const float2 r = cs[c];
      const float a = to_f32(src[2 * c]), b = to_f32(src[2 * c + 1]);
      put(dst[2 * c], a * r.x - b * r.y);
      put(dst[2 * c + 1], b * r.x + a * r.y);
    } else if constexpr (INTER) {
      Chunk<T, VEC> v;
      v.load(src + c * VEC);
#pragma unroll
      for (int k = 0; k < VEC / 2; ++k) {
        const float2 r = cs[c * (VEC / 2) + k];
        const float a = to_f32(v.v[2 * k]), b = to_f32(v.v[2 * k + 1]);
        put(v.v[2 * k], a * r.x - b * r.y);
        put(v.v[2 * k + 1], b * r.x + a * r.y);
      }
      v.store(dst + c * VEC);
    } else {
      Chunk<T, VEC> va, vb;
      va.load(src + c * VEC);
      vb.load(src + pairs + c * VEC);
#pragma unroll
      for (int k = 0; k < VEC; ++k) {
        const float2 r = cs[c * VEC + k];
        const float a = to_f32(va.v[k]), b = to_f32(vb.v[k]);
        put(va.v[k], a * r.x - b * r.y);
        put(vb.v[k], b * r.x + a * r.y);
      }
      va.store(dst + c * VEC);
      vb.store(dst + pairs + c * VEC);
    }
  }
}

}  // namespace

}  // namespace i4tc

using namespace i4tc;

extern "C" int i4tc_rope(const i4tc_rope_args* a, int device, void* stream) {
  I4TC_REQUIRE(a != nullptr, I4TC_EINVAL, "null pointer");
  const void *x = a->x, *positions = a->positions;
  void* out = a->out;
  const int64_t dtype = a->dtype, tokens = a->tokens, heads = a->heads, D = a->D, R = a->R, x_token = a->x_token, x_head = a->x_head,
                out_token = a->out_token, out_head = a->out_head;
  const double* freqs = a->freqs;
  const bool long_positions = a->long_positions != 0, interleaved = a->interleaved != 0;
  I4TC_REQUIRE(dtype == I4TC_BF16 || dtype == I4TC_FP16, I4TC_EUNSUPPORTED, "x must be bfloat16 or float16");
  I4TC_REQUIRE(tokens >= 0 && heads >= 0 && D >= 0 && R >= 0 && R % 2 == 0 && R <= D, I4TC_EINVAL,
               "the rotated part must be an even number of elements of a head");
  if (tokens == 0 || heads == 0 || D == 0) return I4TC_OK;
  I4TC_REQUIRE(tokens < (1ll << 31) && heads <= 65536 && D <= 2048, I4TC_EINVAL, "bad size");
  I4TC_REQUIRE(x && out && (R == 0 || (positions && freqs)), I4TC_EINVAL, "null pointer");
  I4TC_REQUIRE(aligned_to(x, 2) && aligned_to(out, 2) && aligned_to(freqs, 8) && aligned_to(positions, long_positions ? 8 : 4), I4TC_EALIGN,
               "operands must be aligned to their element size");
  const bool in_place = x == out;
  I4TC_REQUIRE(!in_place || (x_token == out_token && x_head == out_head), I4TC_EINVAL, "in place needs the same strides");
  if (in_place && R == 0) return I4TC_OK;
  DeviceGuard guard(device);
  I4TC_CUDA(guard.err);
  RopeParams p = {};
  p.x = x; p.out = out; p.x_token = x_token; p.x_head = x_head; p.out_token = out_token; p.out_head = out_head;
  p.positions = positions; p.freqs = freqs; p.tokens = (int)tokens; p.heads = (int)heads; p.D = (int)D; p.R = (int)R;
  p.scale = (float)a->scale; p.long_positions = long_positions; p.inverse = a->inverse != 0; p.in_place = in_place;
  // the widest access that strides, parts and addresses are multiples of
  int vec = 8;
  const int64_t all = (interleaved ? R : R / 2) | (in_place ? 0 : D - R) | x_token | x_head | out_token | out_head;
  while (vec > 1 && (all % vec != 0 || !aligned_to(x, 2 * vec) || !aligned_to(out, 2 * vec))) vec /= 2;
  // A block takes the tokens and heads that give each thread a few accesses; few tokens are shared out by heads.
  const int64_t accesses = (R / 2 + (in_place ? 0 : D - R)) / vec + 1;
  p.tokens_each = 1;
  while (p.tokens_each < 8 && p.tokens_each * 2 * (R / 2) <= 512 && p.tokens_each * heads * accesses < 4 * kRopeThreads &&
         tokens / (p.tokens_each * 2) >= 8 * 148)
    p.tokens_each *= 2;
  p.heads_each = (int)heads;
  const int64_t blocks = (tokens + p.tokens_each - 1) / p.tokens_each;
  while (p.heads_each > 1 && blocks * ((heads + p.heads_each - 1) / p.heads_each) < 148 && p.heads_each * accesses > kRopeThreads / 2)
    p.heads_each = (p.heads_each + 1) / 2;
  const dim3 grid((unsigned)blocks, (unsigned)((heads + p.heads_each - 1) / p.heads_each));
  const size_t smem = (size_t)p.tokens_each * (R / 2) * sizeof(float2);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto pick = [&](auto type, auto inter) {
    using T = decltype(type);
    constexpr bool INTER = decltype(inter)::value;
    auto kernel = vec == 8   ? rope_kernel<T, 8, INTER>
                  : vec == 4 ? rope_kernel<T, 4, INTER>
                  : vec == 2 ? rope_kernel<T, 2, INTER>
                             : rope_kernel<T, 1, INTER>;
    return launch_kernel(true, kernel, grid, kRopeThreads, smem, st, p);
  };
  I4TC_CUDA(dtype == I4TC_BF16 ? (interleaved ? pick(__nv_bfloat16{}, std::true_type{}) : pick(__nv_bfloat16{}, std::false_type{}))
                               : (interleaved ? pick(__half{}, std::true_type{}) : pick(__half{}, std::false_type{})));
  return I4TC_OK;
}
