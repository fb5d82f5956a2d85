// Keys and values into a paged cache of 4 bits (cache4.h says how it holds them).
//
// Eight elements a lane, so a vector of D takes D / 8 lanes (up to a power of two) and a wave takes several; lowest and highest
// element by exchanges between these lanes. Two bytes an element in, half a byte out: what counts is that loads are 16 bytes. A value's
// byte holds elements 16 apart, which lie two lanes apart: each of the two lanes writes half of the bytes they make.
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
  int tokens, heads, dim, page_size;
};

template <typename T, int LANES>
__global__ __launch_bounds__(256) void store4_kernel(Store4Args a) {
  const int lane = threadIdx.x & 63, part = lane & (LANES - 1);
  const int64_t vector = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int per = 2 * a.heads;
  const int token = (int)(vector / per), which = (int)(vector - (int64_t)token * per);
  const bool value = which >= a.heads;
  const int head = value ? which - a.heads : which;
  const int64_t slot = token < a.tokens ? a.slots[token] : -1;
  const bool here = slot >= 0 && slot < a.num_slots, mine = here && 8 * part < a.dim;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.f;
  float low = INFINITY, high = -INFINITY;
  bool bad = false;
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
      bad |= !(fabsf(x[e]) < INFINITY);
    }
  }
#pragma unroll
  for (int d = LANES / 2; d > 0; d /= 2) low = fminf(low, __shfl_xor(low, d)), high = fmaxf(high, __shfl_xor(high, d));
  const uint64_t odd = __builtin_amdgcn_ballot_w64(bad);
  constexpr uint64_t GROUP = LANES == 64 ? ~0ull : (1ull << LANES) - 1;
  bool broken = (odd >> (lane & ~(LANES - 1)) & GROUP) != 0;
  const bf16_t lo16 = (bf16_t)low;
  const float lo = (float)lo16;
  const bf16_t step16 = (bf16_t)((high - lo) / 15.0f);
  const float step = (float)step16;
  broken |= !(step < INFINITY);
  unsigned codes = 0;
  if (!broken && step > 0.f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) codes |= (unsigned)fminf(fmaxf(rintf((x[e] - lo) / step), 0.f), 15.f) << (4 * e);
  }
  const unsigned others = __shfl_xor(codes, 2);  // the elements 16 further, or before
  if (!mine) return;
  const int64_t page = slot / a.page_size;
  const int off = (int)(slot - page * a.page_size);
  const int64_t row = (page * a.heads + head) * a.page_size + off;  // of this token and head
  if (part == 0) {
    const unsigned pair = broken ? 0x7fc0u : (unsigned)__builtin_bit_cast(unsigned short, lo16) |
                                                 (step > 0.f ? (unsigned)__builtin_bit_cast(unsigned short, step16) << 16 : 0u);
    a.steps[2 * row + value] = pair;
  }
  if (!value) {
    *(unsigned*)(a.k_pages + row * (a.dim / 2) + 4 * part) = codes;
  } else {
    const int w = part >> 2, upper = part >> 1 & 1, words = a.dim / 32;
    const unsigned lows = upper ? others : codes, highs = upper ? codes : others;
    uint8_t* four = a.v_pages + (row - (off & 3)) * (a.dim / 2) + (off & 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int e = 4 * upper + i, c = 8 * (part & 1) + e;
      four[(c * words + w) * 4] = (uint8_t)((lows >> (4 * e) & 15) | (highs >> (4 * e) & 15) << 4);
    }
  }
}

// k, v [tokens, heads, dim] with their tokens k_stride and v_stride elements apart; slots[t] = page * page_size + offset, tokens whose
// slot is in no page are left out.
extern "C" int qrt_store4(const void* k, const void* v, int dtype, int64_t k_stride, int64_t v_stride, void* k_pages, void* v_pages, void* steps,
                          const int* slots, int64_t num_pages, int tokens, int heads, int dim, int page_size, hipStream_t stream) {
  QRT_CHECK(dtype == QRT_BF16 || dtype == QRT_F32, "store4: unknown dtype %d", dtype);
  QRT_CHECK(tokens >= 0 && heads > 0 && num_pages >= 0, "store4: bad sizes tokens=%d heads=%d", tokens, heads);
  QRT_CHECK(dim >= 32 && dim <= 256 && dim % 32 == 0, "store4: heads of 32 to 256 in steps of 32, not %d", dim);
  QRT_CHECK(page_size >= 4 && page_size % 4 == 0, "store4: pages of a multiple of 4 tokens, not %d", page_size);
  const int align = dtype == QRT_BF16 ? 8 : 4;
  QRT_CHECK(((uintptr_t)k | (uintptr_t)v) % 16 == 0 && k_stride % align == 0 && v_stride % align == 0, "store4: rows must begin at multiples of 16 bytes");
  QRT_CHECK(((uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)steps) % 16 == 0, "store4: pages must begin at multiples of 16 bytes");
  if (tokens == 0) return 0;
  const Store4Args a{k, v, (uint8_t*)k_pages, (uint8_t*)v_pages, (unsigned*)steps, slots, k_stride, v_stride, num_pages * page_size, tokens, heads, dim, page_size};
  const int lanes = dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  const int64_t blocks = ((int64_t)tokens * heads * 2 * lanes + 255) / 256;
  QRT_CHECK(blocks < (1ll << 31), "store4: too many tokens for one launch (%d)", tokens);
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
