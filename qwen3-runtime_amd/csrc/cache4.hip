// Keys and values into a paged cache of 4 bits (cache4.h says how it holds them).
//
// Eight elements a lane, so a vector of D takes D / 8 lanes (up to a power of two) and a wave takes several; lowest and highest
// element by exchanges between these lanes. Two bytes an element in, half a byte out: what counts is that loads are 16 bytes. A value's
// byte holds elements 16 apart, which lie two lanes apart: each of the two lanes writes half of the bytes they make.
// 2,047 tokens of 8 heads of 128, 10.8 MB in and out: 6.0 us, 1.8 TB/s; 8 tokens 2.8 us, a launch. Of many tokens a launch and the way of one load bound it: a wave
// takes four vectors and ends, and waits in 54 % of its time; its 290 vector instructions take 28 % of the SIMDs' cycles. It was 8.0 us with divisions of
// 64-bit numbers and of every element, and exchanges through LDS.
#include "common.h"
#include "cache4.h"

struct Store4Args {
  const void* k;
  const void* v;
  uint8_t* k_pages;
  uint8_t* v_pages;
  unsigned* steps;  // pairs of bfloat16
  const int* slots;
  int64_t k_stride, v_stride;  // elements from token to token
  int64_t num_slots;
  int tokens, heads, dim;
  PageMagic page, vectors;  // division by the page size, and by the vectors (or heads) of a token
};

// codes = clamp(rint((x - lo) / step), 0, 15) with the quotient rounded to float32 first. From the rounded reciprocal of the step a product, its remainder
// and a correction give that quotient (Markstein's: the remainder is exact, the corrected quotient rounded as a division's would be) in three
// instructions an element for some ten, as long as nothing leaves the normal range: steps under 2^-60, whose remainders might, divide.
struct Coder {
  float lo, step, by;
  bool divides;  // a lane of the wave has to
  __device__ __forceinline__ Coder(float lo, float step) : lo(lo), step(step), by(1.0f / step), divides(__builtin_amdgcn_ballot_w64(step < 0x1p-60f) != 0) {}
  __device__ __forceinline__ unsigned code(float quotient) const { return (unsigned)fminf(fmaxf(rintf(quotient), 0.f), 15.f); }
  template <int N>
  __device__ __forceinline__ void operator()(const float (&x)[N], unsigned (&codes)[N]) const {
    if (divides) {
#pragma unroll
      for (int e = 0; e < N; ++e) codes[e] = code((x[e] - lo) / step);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float above = x[e] - lo, near = above * by;
        codes[e] = code(fmaf(fmaf(-near, step, above), by, near));
      }
    }
  }
};

template <int CTRL>
__device__ __forceinline__ unsigned moved(unsigned x) { return (unsigned)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, false); }
constexpr int BY_ONE = 0xb1, BY_TWO = 0x4e, HALF_MIRROR = 0x141, MIRROR = 0x140;  // lanes change places in fours, eights, sixteens
template <int CTRL>
__device__ __forceinline__ void meet(float& low, float& high) {
  low = fminf(low, __uint_as_float(moved<CTRL>(__float_as_uint(low)))), high = fmaxf(high, __uint_as_float(moved<CTRL>(__float_as_uint(high))));
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void store4_kernel(Store4Args a) {
  const int lane = threadIdx.x & 63, part = lane & (LANES - 1);
  int token, which;
  page_of(a.vectors, blockIdx.x * (256 / LANES) + threadIdx.x / LANES, token, which);
  const bool value = which >= a.heads;
  const int head = value ? which - a.heads : which;
  const int64_t slot = token < a.tokens ? a.slots[token] : -1;
  const bool here = slot >= 0 && slot < a.num_slots, mine = here && 8 * part < a.dim;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  float low = INFINITY, high = -INFINITY;
  float odd = 0.f;  // NaN from the first infinity or NaN on
  if (mine) {
    const T* src = (const T*)(value ? a.v : a.k) + token * (value ? a.v_stride : a.k_stride) + head * a.dim + 8 * part;
    if constexpr (sizeof(T) == 2) {
      const bf16x8_t y = *(const bf16x8_t*)src;
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)y[e];
    } else {
      const f32x4_t y = *(const f32x4_t*)src, z = *(const f32x4_t*)(src + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = y[e], x[4 + e] = z[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      low = fminf(low, x[e]), high = fmaxf(high, x[e]);
      odd = fmaf(x[e], 0.f, odd);
    }
  }
  meet<BY_ONE>(low, high), meet<BY_TWO>(low, high);
  if constexpr (LANES > 4) meet<HALF_MIRROR>(low, high);
  if constexpr (LANES > 8) meet<MIRROR>(low, high);
  if constexpr (LANES > 16) low = fminf(low, __shfl_xor(low, 16)), high = fmaxf(high, __shfl_xor(high, 16));
  const uint64_t bad = __builtin_amdgcn_ballot_w64(odd != odd);
  constexpr uint64_t GROUP = LANES == 64 ? ~0ull : (1ull << LANES) - 1;
  bool broken = (bad >> (lane & ~(LANES - 1)) & GROUP) != 0;
  const bf16_t lo16 = (bf16_t)low;
  const float lo = (float)lo16;
  const bf16_t step16 = (bf16_t)((high - lo) / 15.0f);
  const float step = (float)step16;
  broken |= !(step < INFINITY);
  unsigned codes = 0;
  if (!broken && step > 0.f) {
    unsigned each[8];
    Coder(lo, step)(x, each);
#pragma unroll
    for (int e = 0; e < 8; ++e) codes |= each[e] << (4 * e);
  }
  const unsigned others = moved<BY_TWO>(codes);  // the elements 16 further, or before
  if (!mine) return;
  int page, off;
  page_of(a.page, (int)slot, page, off);
  const int64_t row = ((int64_t)page * a.heads + head) * (int)a.page.size + off;  // of this token and head
  if (part == 0) {
    const unsigned pair = broken ? 0x7fc0u : (unsigned)__builtin_bit_cast(unsigned short, lo16) |
                                                 (step > 0.f ? (unsigned)__builtin_bit_cast(unsigned short, step16) << 16 : 0u);
    a.steps[2 * row + value] = pair;
  }
  if (!value) {
    *(unsigned*)(a.k_pages + row * (a.dim / 2) + 4 * part) = codes;
  } else {
    const int w = part >> 2, upper = part >> 1 & 1, words = a.dim / 32;
    const unsigned lows = (upper ? others : codes) >> (16 * upper), highs = (upper ? codes : others) >> (16 * upper);
    const unsigned even = (lows & 0x0f0fu) | (highs & 0x0f0fu) << 4, uneven = (lows >> 4 & 0x0f0fu) | (highs & 0xf0f0u);
    uint8_t* to = a.v_pages + (row - (off & 3)) * (a.dim / 2) + (off & 3) + ((8 * (part & 1) + 4 * upper) * words + w) * 4;
    to[0] = (uint8_t)even;
    to[4 * words] = (uint8_t)uneven;
    to[8 * words] = (uint8_t)(even >> 8);
    to[12 * words] = (uint8_t)(uneven >> 8);
  }
}

// Few tokens: q/k norm, rotation, the queries' store and the quantising store of keys and values in one kernel, a wave a head. A lane has
// pairs of elements that turn together, as the rotation of a whole cache has them for few tokens (the same sums, the same bits of the
// queries, keys rounded to the activations' type before they are quantised); codes meet in LDS, a byte an element, to be packed. A decode
// step's store cost a kernel of 3 us more without it.
struct Norm4Args {
  const void* qkv;  // [tokens, stride]: q, k and v heads
  int64_t stride;
  const float* q_weight;  // null: no norm
  const float* k_weight;
  const float* inv_freq;  // null: no rotation
  const int* positions;
  void* q_out;
  int nq, rot_pairs;
  float eps;
};

template <typename T>
__global__ __launch_bounds__(256) void norm_store4_kernel(Norm4Args n, Store4Args a) {
  __shared__ __align__(8) uint8_t codes_of[4][256];
  const int lane = threadIdx.x & 63, wave = uniform_wave_number();
  const int D = a.dim, half = D >> 1, rp = n.rot_pairs;
  int t, h;
  page_of(a.vectors, blockIdx.x * 4 + wave, t, h);
  if (t >= a.tokens) return;
  const bool is_q = h < n.nq, value = h >= n.nq + a.heads;
  const T* src = (const T*)n.qkv + (size_t)t * n.stride + (size_t)h * D;
  const float* w = is_q ? n.q_weight : value ? nullptr : n.k_weight;
  const bool turns = n.inv_freq && !value;
  // pair p: elements p and rp + p where it turns; behind those the others
  auto first_of = [&](int p) { return p < rp ? p : p + rp; };
  auto second_of = [&](int p) { return p < rp ? p + rp : p + half; };
  float x1[2], x2[2], w1[2], w2[2], fr[2];
  float ss = 0.f;
  const float pos = turns ? (float)n.positions[t] : 0.f;
  const int64_t slot = is_q ? 0 : a.slots[t];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = lane + 64 * i;
    x1[i] = x2[i] = fr[i] = 0.f, w1[i] = w2[i] = 1.f;
    if (p < half) {
      x1[i] = to_f32<T>(src[first_of(p)]), x2[i] = to_f32<T>(src[second_of(p)]);
      if (w) w1[i] = w[first_of(p)], w2[i] = w[second_of(p)];
      if (turns && p < rp) fr[i] = n.inv_freq[p];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) ss += x1[i] * x1[i] + x2[i] * x2[i];
  if (w) {
    ss = wave_sum(ss);
    const float inv = rsqrtf(ss / (float)D + n.eps);
#pragma unroll
    for (int i = 0; i < 2; ++i) x1[i] = x1[i] * inv * w1[i], x2[i] = x2[i] * inv * w2[i];
  }
  if (turns) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (lane + 64 * i < rp) {
        float sn, c;
        sincos_angle(pos * fr[i], &sn, &c);
        const float y1 = x1[i] * c - x2[i] * sn, y2 = x2[i] * c + x1[i] * sn;
        x1[i] = y1, x2[i] = y2;
      }
    }
  }
  if (is_q) {
    T* to = (T*)n.q_out + ((size_t)t * n.nq + h) * D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int p = lane + 64 * i;
      if (p < half) to[first_of(p)] = from_f32<T>(x1[i]), to[second_of(p)] = from_f32<T>(x2[i]);
    }
    return;
  }
  float low = INFINITY, high = -INFINITY;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (lane + 64 * i >= half) continue;
    x1[i] = to_f32<T>(from_f32<T>(x1[i])), x2[i] = to_f32<T>(from_f32<T>(x2[i]));
    low = fminf(low, fminf(x1[i], x2[i])), high = fmaxf(high, fmaxf(x1[i], x2[i]));
    bad |= !(fabsf(x1[i]) < INFINITY) || !(fabsf(x2[i]) < INFINITY);
  }
  bool broken = __builtin_amdgcn_ballot_w64(bad) != 0;
  high = wave_max(high), low = -wave_max(-low);
  const bf16_t lo16 = (bf16_t)low;
  const float lo = (float)lo16;
  const bf16_t step16 = (bf16_t)((high - lo) / 15.0f);
  const float step = (float)step16;
  broken |= !(step < INFINITY);
  const bool flat = broken || !(step > 0.f);
  unsigned codes1[2], codes2[2];
  const Coder coder(lo, flat ? 1.f : step);
  coder(x1, codes1), coder(x2, codes2);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int p = lane + 64 * i;
    if (p < half) {
      codes_of[wave][first_of(p)] = flat ? 0 : (uint8_t)codes1[i];
      codes_of[wave][second_of(p)] = flat ? 0 : (uint8_t)codes2[i];
    }
  }
  __builtin_amdgcn_wave_barrier();  // a wave's reads of LDS come behind its writes
  if (slot < 0 || slot >= a.num_slots) return;
  const int head = h - n.nq - (value ? a.heads : 0);
  int page, off;
  page_of(a.page, (int)slot, page, off);
  const int64_t row = ((int64_t)page * a.heads + head) * (int)a.page.size + off;
  if (lane == 0) {
    a.steps[2 * row + value] = broken ? 0x7fc0u : (unsigned)__builtin_bit_cast(unsigned short, lo16) | (flat ? 0u : (unsigned)__builtin_bit_cast(unsigned short, step16) << 16);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int b = lane + 64 * i;  // a byte of D / 2
    if (b >= half) continue;
    if (!value) {
      a.k_pages[row * half + b] = codes_of[wave][2 * b] | codes_of[wave][2 * b + 1] << 4;
    } else {
      const int words = D / 32, c = b / words, e = 32 * (b - c * words) + c;
      a.v_pages[(row - (off & 3)) * half + 4 * b + (off & 3)] = codes_of[wave][e] | codes_of[wave][e + 16] << 4;
    }
  }
}

static int check_store4(int dtype, int64_t num_pages, int tokens, int heads, int dim, int page_size, const void* k_pages, const void* v_pages, const void* steps) {
  QRT_CHECK(dtype == QRT_BF16 || dtype == QRT_F32, "store4: unknown dtype %d", dtype);
  QRT_CHECK(tokens >= 0 && heads > 0 && num_pages >= 0, "store4: bad sizes tokens=%d heads=%d", tokens, heads);
  QRT_CHECK(dim >= 32 && dim <= 256 && dim % 32 == 0, "store4: heads of 32 to 256 in steps of 32, not %d", dim);
  QRT_CHECK(page_size >= 4 && page_size % 4 == 0, "store4: pages of a multiple of 4 tokens, not %d", page_size);
  QRT_CHECK(((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)steps) % 16 == 0, "store4: pages must begin at multiples of 16 bytes");
  return 0;
}

// qkv [tokens, stride]: nq heads of queries, nkv of keys and nkv of values. Weights may be null (no norm), inv_freq too (no rotation; otherwise rot_pairs
// frequencies). q_out [tokens, nq, dim]. Tokens whose slot is in no page store nothing.
extern "C" int qrt_norm_store4(const void* qkv, int dtype, int64_t stride, const float* q_weight, const float* k_weight, float eps, const float* inv_freq,
                               const int* positions, int rot_pairs, void* q_out, void* k_pages, void* v_pages, void* steps, const int* slots, int64_t num_pages,
                               int tokens, int nq, int nkv, int dim, int page_size, hipStream_t stream) {
  if (check_store4(dtype, num_pages, tokens, nkv, dim, page_size, k_pages, v_pages, steps)) return -1;
  QRT_CHECK(nq > 0 && stride >= (int64_t)(nq + 2 * nkv) * dim, "norm_store4: rows of %lld for %d + 2 * %d heads of %d", (long long)stride, nq, nkv, dim);
  QRT_CHECK(!inv_freq || (positions && rot_pairs >= 1 && rot_pairs <= dim / 2), "norm_store4: %d pairs turn in heads of %d", rot_pairs, dim);
  QRT_CHECK((int64_t)tokens * (nq + 2 * nkv) < (1ll << 31), "norm_store4: too many tokens for one launch (%d)", tokens);
  if (tokens == 0) return 0;
  const Norm4Args n{qkv, stride, q_weight, k_weight, inv_freq, positions, q_out, nq, inv_freq ? rot_pairs : dim / 2, eps};
  const Store4Args a{nullptr, nullptr, (uint8_t*)k_pages, (uint8_t*)v_pages, (unsigned*)steps, slots, 0, 0, num_pages * page_size, tokens, nkv, dim, page_magic(page_size), page_magic(nq + 2 * nkv)};
  const int blocks = (tokens * (nq + 2 * nkv) + 3) / 4;
  if (dtype == QRT_BF16) norm_store4_kernel<bf16_t><<<blocks, 256, 0, stream>>>(n, a);
  else norm_store4_kernel<float><<<blocks, 256, 0, stream>>>(n, a);
  QRT_LAUNCH_CHECK("norm_store4");
  return 0;
}

// k, v [tokens, heads, dim] with their tokens k_stride and v_stride elements apart; slots[t] = page * page_size + offset, tokens whose
// slot is in no page are left out.
extern "C" int qrt_store4(const void* k, const void* v, int dtype, int64_t k_stride, int64_t v_stride, void* k_pages, void* v_pages, void* steps,
                          const int* slots, int64_t num_pages, int tokens, int heads, int dim, int page_size, hipStream_t stream) {
  if (check_store4(dtype, num_pages, tokens, heads, dim, page_size, k_pages, v_pages, steps)) return -1;
  const int align = dtype == QRT_BF16 ? 8 : 4;
  QRT_CHECK(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_stride % align == 0 && v_stride % align == 0, "store4: rows must begin at multiples of 16 bytes");
  if (tokens == 0) return 0;
  const Store4Args a{k, v, (uint8_t*)k_pages, (uint8_t*)v_pages, (unsigned*)steps, slots, k_stride, v_stride, num_pages * page_size, tokens, heads, dim, page_magic(page_size), page_magic(2 * heads)};
  const int lanes = dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  const int64_t blocks = ((int64_t)tokens * heads * 2 * lanes + 255) / 256;
  QRT_CHECK(blocks * (256 / lanes) < (1ll << 31), "store4: too many tokens for one launch (%d)", tokens);
#define GO(L)                                                                                     \
  do {                                                                                            \
    if (dtype == QRT_BF16) store4_kernel<bf16_t, L><<<(unsigned)blocks, 256, 0, stream>>>(a);     \
    else store4_kernel<float, L><<<(unsigned)blocks, 256, 0, stream>>>(a);                        \
  } while (0)
  if (lanes == 4) GO(4);
  else if (lanes == 8) GO(8);
  else if (lanes == 16) GO(16);
  else GO(32);
#undef GO
  QRT_LAUNCH_CHECK("store4");
  return 0;
}
