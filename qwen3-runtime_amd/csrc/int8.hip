// Rows to 8-bit integers, and the product of up to 64 such rows with a weight of 8-bit integers.
//
// quantize_rows: a row a block (up to 1,024 columns a wave), held in registers between its maximum and its codes, so memory is
// read once: 2 K bytes in, K out. 2,048 rows of 9,728 bfloat16 (60 MB) 11.2 us, 5.3 TB/s; 24 rows 2.7 us, a launch.
//
// int8_rows: few rows stream the weight, which is what bounds them. The MFMA of 16 x 16 x 64 takes 16 bytes of a row a lane, and
// direct loads bring 8 rows x 128 bytes, whole lines, as for bfloat16: the bytes lie alike, two k-steps are 128 columns. A
// block owns 8, 16 or 32 weight rows and all of K, its waves take the steps of 128 columns round-robin, each with a ring of its
// own, and their whole sums meet in LDS; the order of whole sums does not matter. Eight weight rows a block (the operand's other eight
// repeat them) leave the busiest compute unit less to fetch where there are few. Weights from memory, us and TB/s: 1 row by 6,144 x 2,560 4.6, 3.4
// with the row's codes; 24 rows by 2,560 x 9,728 7.7, 3.2 (160 blocks for 256 compute units: more and shorter ones of 8 weight rows took
// longer), by 6,144 x 4,096 8.2, 3.1 (384 blocks: 32 weight rows for the busiest unit, 24 on average); gated, 8 rows by 2 x 9,728 x 2,560 9.8, 5.1. A launch and the first bytes' way are some 2.5 us of each.
#include "common.h"
#include "direct.h"
#include "gemm_epilogue.h"
#include "int8.h"

// ---------------------------------------------------------------- rows to codes

template <typename T, bool ALIGNED>
__device__ __forceinline__ void load_row8(const T* __restrict__ row, int at, int K, float (&v)[8]) {
  if (ALIGNED) {
    if (at < K) {  // K is a multiple of 8 then
      if constexpr (sizeof(T) == 2) {
        const bf16x8_t x = *(const bf16x8_t*)(row + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)x[e];
      } else {
        const f32x4_t x = *(const f32x4_t*)(row + at), y = *(const f32x4_t*)(row + at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[e], v[4 + e] = y[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = at + e < K ? to_f32<T>(row[at + e]) : 0.f;
  }
}

// THREADS to a row (64, or a whole block); KEEP pieces of 8 columns a thread stay in registers, wider rows are read a second time.
template <typename T, int THREADS, int KEEP, bool ALIGNED>
__global__ __launch_bounds__(THREADS > 256 ? THREADS : 256) void quantize_rows_kernel(const T* __restrict__ x, int8_t* __restrict__ codes, float* __restrict__ scale, int M, int K, int width) {
  constexpr int WAVES = THREADS / 64;
  __shared__ unsigned part[WAVES];
  const int t = threadIdx.x % THREADS;
  const int row = THREADS < 256 ? blockIdx.x * (256 / THREADS) + threadIdx.x / THREADS : blockIdx.x;
  const T* src = x + (size_t)min(row, M - 1) * K;
  float v[KEEP][8];
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) load_row8<T, ALIGNED>(src, 8 * (t + THREADS * i), K, v[i]);
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(v[i][e]));
  for (int at = 8 * (t + THREADS * KEEP); at < K; at += 8 * THREADS) {
    float w[8];
    load_row8<T, ALIGNED>(src, at, K, w);
#pragma unroll
    for (int e = 0; e < 8; ++e) most = max(most, magnitude_bits(w[e]));
  }
  most = wave_max_bits(most);
  if (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
    __syncthreads();
    most = part[0];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) most = max(most, part[i]);
  }
  if (row >= M) return;
  const float by = code_factor(most);
  int8_t* out = codes + (size_t)row * width;
  auto store = [&](int at, const float (&w)[8]) {
    typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
    *(u32x2_t*)(out + at) = (u32x2_t){codes4(w[0], w[1], w[2], w[3], by), codes4(w[4], w[5], w[6], w[7], by)};
  };
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int at = 8 * (t + THREADS * i);
    if (at < width) store(at, v[i]);
  }
  for (int at = 8 * (t + THREADS * KEEP); at < width; at += 8 * THREADS) {
    float w[8];
    load_row8<T, ALIGNED>(src, at, K, w);
    store(at, w);
  }
  if (t == 0) scale[row] = row_scale_of(most);
}

template <typename T>
static void launch_quantize(const T* x, int8_t* codes, float* scale, int M, int K, int width, hipStream_t stream) {
  const bool aligned = K % 8 == 0 && (uintptr_t)x % 16 == 0;
#define GO(THREADS, KEEP, ALIGNED)                                                                                                     \
  quantize_rows_kernel<T, THREADS, KEEP, ALIGNED>                                                                                      \
      <<<dim3(THREADS < 256 ? (M + 256 / THREADS - 1) / (256 / THREADS) : M), dim3(THREADS < 256 ? 256 : THREADS), 0, stream>>>(x, codes, scale, M, K, width)
  // a wave a row needs no barrier: 1,999 rows of 2,560 columns 6.8 -> 4.2 us. Few long rows leave most compute units idle and are over as
  // soon as one of them is: 1,024 threads.
  if (!aligned) GO(256, 4, false);
  else if (width <= 1024) GO(64, 2, true);
  else if (width <= 4096 && M >= 512) GO(64, 8, true);
  else if (width <= 4096) GO(256, 2, true);
  else if (M < 256) GO(1024, 2, true);
  else GO(256, 5, true);
#undef GO
}

static int check_width(const char* name, int M, int K, int width) {
  QRT_CHECK(M >= 0 && K > 0 && width >= K && width % INT8_STAGE == 0 && width <= INT8_MOST_WIDTH, "%s: bad sizes M=%d K=%d, rows of %d", name, M, K, width);
  return 0;
}

// codes [M, width] (columns K and on are zeros), scale [M]; width: K up to a multiple of 128
extern "C" int qrt_quantize_rows(const void* x, int dtype, void* codes, float* scale, int M, int K, int width, hipStream_t stream) {
  if (check_width("quantize_rows", M, K, width)) return -1;
  QRT_CHECK(dtype == QRT_BF16 || dtype == QRT_F32, "quantize_rows: unknown dtype %d", dtype);
  QRT_CHECK((uintptr_t)codes % 16 == 0, "quantize_rows: codes must begin at a multiple of 16 bytes");
  if (M == 0) return 0;
  if (dtype == QRT_BF16) launch_quantize((const bf16_t*)x, (int8_t*)codes, scale, M, K, width, stream);
  else launch_quantize((const float*)x, (int8_t*)codes, scale, M, K, width, stream);
  QRT_LAUNCH_CHECK("quantize_rows");
  return 0;
}

// ---------------------------------------------------------------- a norm's rows as codes

// residual += delta (or the sum of its planes, in their order), and the codes of the row's RMS norm, which is rounded to bfloat16 before where
// the activations are: what add_rmsnorm and quantize_rows make, without the row between them. A block a row, all of it in registers.
template <typename TD, int KEEP, bool ROUND>
__global__ __launch_bounds__(256) void add_rmsnorm_codes_kernel(float* __restrict__ residual, const TD* __restrict__ delta, const float* __restrict__ weight,
                                                                int8_t* __restrict__ codes, float* __restrict__ scale, int hidden, int width, float eps,
                                                                int planes, size_t plane_stride) {
  constexpr int AHEAD = KEEP > 4 ? 2 : 4;
  __shared__ float red[16];
  __shared__ unsigned part[4];
  float* x = residual + (size_t)blockIdx.x * hidden;
  const TD* d = delta + (size_t)blockIdx.x * hidden;
  f32x4_t v[KEEP], w[KEEP];
  float squares = 0.f;
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int at = min(4 * ((int)threadIdx.x + 256 * i), hidden - 4);
    v[i] = *(const f32x4_t*)(x + at), w[i] = *(const f32x4_t*)(weight + at);
  }
  typedef TD dvec_t __attribute__((ext_vector_type(4)));
  for (int p = 0; p < planes; p += AHEAD) {  // a load that waits for the one before costs a microsecond
    dvec_t y[AHEAD][KEEP];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q)
#pragma unroll
      for (int i = 0; i < KEEP; ++i)
        y[q][i] = *(const dvec_t*)(d + min(p + q, planes - 1) * plane_stride + min(4 * ((int)threadIdx.x + 256 * i), hidden - 4));
#pragma unroll
    for (int q = 0; q < AHEAD; ++q)
      if (p + q < planes)
#pragma unroll
        for (int i = 0; i < KEEP; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][e] += to_f32<TD>(y[q][i][e]);
  }
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int at = 4 * ((int)threadIdx.x + 256 * i);
    if (at >= hidden) v[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    else if (planes > 0) *(f32x4_t*)(x + at) = v[i];
    squares += (v[i][0] * v[i][0] + v[i][1] * v[i][1]) + (v[i][2] * v[i][2] + v[i][3] * v[i][3]);
  }
  const float by = rsqrtf(block_sum(squares, red) / (float)hidden + eps);
  unsigned most = 0;
#pragma unroll
  for (int i = 0; i < KEEP; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[i][e] = v[i][e] * by * w[i][e];
      if (ROUND) v[i][e] = (float)(bf16_t)v[i][e];
      most = max(most, magnitude_bits(v[i][e]));
    }
  most = wave_max_bits(most);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = most;
  __syncthreads();
  most = max(max(part[0], part[1]), max(part[2], part[3]));
  const float factor = code_factor(most);
#pragma unroll
  for (int i = 0; i < KEEP; ++i) {
    const int at = 4 * ((int)threadIdx.x + 256 * i);
    if (at < width) *(unsigned*)(codes + (size_t)blockIdx.x * width + at) = codes4(v[i][0], v[i][1], v[i][2], v[i][3], factor);
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = row_scale_of(most);
}

// Rows of up to 8,192 columns, a multiple of 4. delta may be null (planes 0).
extern "C" int qrt_add_rmsnorm_codes(float* residual, const void* delta, int delta_dtype, const float* weight, void* codes, float* scale, int rows, int hidden,
                                     int width, float eps, int planes, int64_t plane_stride, int round, hipStream_t stream) {
  if (check_width("add_rmsnorm_codes", rows, hidden, width)) return -1;
  QRT_CHECK(hidden % 4 == 0 && width <= 8192, "add_rmsnorm_codes: rows of %d", hidden);
  QRT_CHECK(planes >= 0 && (planes == 0 || delta), "add_rmsnorm_codes: %d planes", planes);
  QRT_CHECK(delta_dtype == QRT_BF16 || delta_dtype == QRT_F32, "add_rmsnorm_codes: unknown dtype %d", delta_dtype);
  QRT_CHECK(((uintptr_t)residual | (uintptr_t)delta | (uintptr_t)weight | (uintptr_t)codes) % 16 == 0, "add_rmsnorm_codes: rows must begin at multiples of 16 bytes");
  if (rows == 0) return 0;
#define GO(TD, KEEP, ROUND) \
  add_rmsnorm_codes_kernel<TD, KEEP, ROUND><<<rows, 256, 0, stream>>>(residual, (const TD*)delta, weight, (int8_t*)codes, scale, hidden, width, eps, planes, plane_stride)
#define BY_WIDTH(TD, ROUND)                    \
  do {                                         \
    if (width <= 1024) GO(TD, 1, ROUND);       \
    else if (width <= 2048) GO(TD, 2, ROUND);  \
    else if (width <= 4096) GO(TD, 4, ROUND);  \
    else GO(TD, 8, ROUND);                     \
  } while (0)
  if (delta_dtype == QRT_BF16) {
    if (round) BY_WIDTH(bf16_t, true);
    else BY_WIDTH(bf16_t, false);
  } else {
    if (round) BY_WIDTH(float, true);
    else BY_WIDTH(float, false);
  }
#undef BY_WIDTH
#undef GO
  QRT_LAUNCH_CHECK("add_rmsnorm_codes");
  return 0;
}

// ---------------------------------------------------------------- few rows

struct Int8Rows {
  const void* x;        // FUSED: rows as they are [M, K]
  const int8_t* a;      // otherwise their codes [M, width] and scales [M]
  const float* a_scale;
  const int8_t* w;      // [N or 2 N, width]
  const float* w_scale;
  void* c;
  int M, N, K, width;
  GatedEpilogue ep;
};

// Rows that a block turns into codes itself (FUSED): up to eight, one or two to each of its four waves, or one to two or all four of them; a
// lane has ITS pieces of 8 columns of each, in registers from the loads to the codes. Every block does so again, so it pays while blocks and rows are few: us
// with a kernel in front and fused at 1 and 4 rows 6,144 x 2,560 7.0, 7.1 and 4.5, 5.2; 6,144 x 4,096 9.0, 9.1 and 6.0, 6.5; gated, 9,728 x 2,560
// (1,216 blocks) 12.0, 12.1 and 11.7, 13.7, 12,288 x 4,096 (1,536) 18.5, 18.6 and 21.3, 24.1.
// Five to eight rows of 1,024 columns 4.0 to 4.1 fused by 2,560 outputs and some 4.7 not, of 2,560 columns 6.5 and 5.9; 16 rows of 1,024 5.8 and 5.1.
constexpr int FUSED_MOST = 10;
constexpr int fused_parts(int M) { return M == 1 ? 4 : M == 2 ? 2 : 1; }
constexpr int fused_its(int M, int width) { return (width / 8 + 64 * fused_parts(M) - 1) / (64 * fused_parts(M)); }
constexpr bool fused_takes(int M, int N, int width) {
  return M >= 1 && (M <= 4 ? N <= 8 * 1100 && fused_its(M, width) <= FUSED_MOST : M <= 8 && N <= 4096 && fused_its(M, width) <= 2);
}

// NW waves; WU units of eight weight rows (1: the operand's rows 8 to 15 repeat the others); MB blocks of 16 rows of the
// activations (FEW: eight); GATED: half of the units are gate rows, half the up rows that belong to them.
// ITS > 0: FUSED, ROWS rows of the activations a wave (or a part of one).
template <int NW, int WU, int MB, bool FEW, int U, bool GATED, int ROWS, int ITS, typename TX, typename TO>
__global__ __launch_bounds__(64 * NW) void int8_rows_kernel(Int8Rows p) {
  constexpr bool FUSED = ITS > 0;
  constexpr int NT = WU == 1 ? 1 : WU / 2, AU = FEW ? 1 : 2 * MB, LOADS = WU + (FUSED ? 0 : AU), SLOT = LOADS * 1024;
  constexpr int OUTS = GATED ? 4 * WU : 8 * WU, ONCE = 2;  // outputs of a block; the cache policy of a non-temporal load
  static_assert((U - 1) * LOADS < 64, "the loads' counter holds 63");
  static_assert(!FUSED || (NW == 4 && FEW), "the waves that share a row are counted for four");
  extern __shared__ __align__(16) unsigned char rows_lds[];  // [NW][U] slots, later the sums; FUSED: the rows' codes behind them
  __shared__ unsigned most_of[FUSED ? 4 * ROWS : 1];
  const int lane = threadIdx.x & 63, wave = uniform_wave_number();
  const int r16 = lane & 15, quad = lane >> 4, sub = lane >> 3, piece = (lane & 7) ^ sub;
  const int n0 = blockIdx.x * OUTS;
  unsigned char* ring = rows_lds + (size_t)wave * U * SLOT;
  constexpr size_t MEET = (size_t)NW * NT * MB * 1024, RINGS = (size_t)NW * U * SLOT;
  unsigned char* const own_codes = rows_lds + (RINGS > MEET ? RINGS : MEET);
  const int width = p.width, steps = width / INT8_STAGE;

  // FUSED: the rows come first, and are waited for behind the weights' loads
  float v[FUSED ? ROWS * ITS : 1][8];
  const int parts = fused_parts(p.M), code_rows = 4 * ROWS / parts, own_row = wave / parts, own_at = 8 * ((wave - own_row * parts) * 64 + lane);
  if constexpr (FUSED) {
#pragma unroll
    for (int k = 0; k < ROWS; ++k)
#pragma unroll
      for (int j = 0; j < ITS; ++j) {
        const int row = own_row + 4 * k;
        load_row8<TX, true>((const TX*)p.x + (size_t)min(row, p.M - 1) * p.K, row < p.M ? own_at + 512 * parts * j : p.K, p.K, v[k * ITS + j]);
      }
  }
  const int8_t* src[LOADS];
#pragma unroll
  for (int u = 0; u < WU; ++u) {  // rows past the end repeat the last; not stored
    const int up = GATED && (WU == 2 ? u == 1 : u >= WU / 2);
    const int unit = GATED ? (WU == 2 ? 0 : u % (WU / 2)) : u;
    src[u] = p.w + (size_t)(min(n0 + 8 * unit + sub, p.N - 1) + (up ? p.N : 0)) * width + 16 * piece;
  }
  if constexpr (!FUSED) {
#pragma unroll
    for (int u = 0; u < AU; ++u) src[WU + u] = p.a + (size_t)min(8 * u + sub, p.M - 1) * width + 16 * piece;
  }
  const int mine = max(0, (steps - wave + NW - 1) / NW);
  auto fetch = [&](int i, int slot) {
    const size_t at = (size_t)(wave + i * NW) * INT8_STAGE;
#pragma unroll
    for (int u = 0; u < LOADS; ++u) {
      if (u < WU) __builtin_amdgcn_global_load_lds((global_ptr_t)(src[u] + at), (lds_ptr_t)(ring + slot * SLOT + u * 1024), 16, 0, ONCE);
      else __builtin_amdgcn_global_load_lds((global_ptr_t)(src[u] + at), (lds_ptr_t)(ring + slot * SLOT + u * 1024), 16, 0, 0);
    }
  };
  int fetched = 0;
  for (; fetched < U && fetched < mine; ++fetched) fetch(fetched, fetched);

  if constexpr (FUSED) {
    __shared__ unsigned part_of[4];
    unsigned most[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      most[k] = 0;
#pragma unroll
      for (int j = 0; j < ITS; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) most[k] = max(most[k], magnitude_bits(v[k * ITS + j][e]));
      most[k] = wave_max_bits(most[k]);
    }
    if (ROWS == 1 && parts > 1) {
      if (lane == 0) part_of[wave] = most[0];
      QRT_WAIT_LDS();
      QRT_BARRIER();
      for (int i = 0; i < parts; ++i) most[0] = max(most[0], part_of[own_row * parts + i]);
    }
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
      const int row = own_row + 4 * k;
      if (row >= p.M) continue;
      if (lane == 0) most_of[row] = most[k];
      const float by = code_factor(most[k]);
#pragma unroll
      for (int j = 0; j < ITS; ++j) {
        const int at = own_at + 512 * parts * j;
        const float(&x)[8] = v[k * ITS + j];
        typedef unsigned u32x2_t __attribute__((ext_vector_type(2)));
        // piece c of 16 columns of a stage's row r lies at 16 (c ^ (r & 7)), as in the rings
        unsigned char* to = own_codes + (size_t)((at >> 7) * code_rows + row) * 128 + 16 * (((at >> 4) & 7) ^ (row & 7)) + (at & 8);
        if (at < width) *(u32x2_t*)to = (u32x2_t){codes4(x[0], x[1], x[2], x[3], by), codes4(x[4], x[5], x[6], x[7], by)};
      }
    }
    QRT_WAIT_LDS();
    QRT_BARRIER();
  }

  i32x4_t acc[NT][MB];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b) acc[t][b] = (i32x4_t){0, 0, 0, 0};
  const int rw = WU == 1 ? r16 & 7 : r16, ra = FUSED ? r16 & (code_rows - 1) : FEW ? r16 & 7 : r16;
  const int w_at[2] = {rw * 128 + 16 * (quad ^ (r16 & 7)), rw * 128 + 16 * ((4 + quad) ^ (r16 & 7))};
  const int a_at[2] = {ra * 128 + 16 * (quad ^ (ra & 7)), ra * 128 + 16 * ((4 + quad) ^ (ra & 7))};
  int slot = 0;
  for (int i = 0; i < mine; ++i) {
    // step i has landed when at most the U - 1 steps fetched after it are still on their way
    if (fetched - i == U) QRT_WAIT_LOADS((U - 1) * LOADS);
    else QRT_WAIT_LOADS(0);
    const unsigned char* at = ring + slot * SLOT;
    const unsigned char* codes = FUSED ? own_codes + (size_t)((wave + i * NW) * code_rows) * 128 : at + WU * 1024;
    i32x4_t w[NT][2], a[MB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int t = 0; t < NT; ++t) w[t][h] = *(const i32x4_t*)(at + t * 2048 + w_at[h]);
#pragma unroll
      for (int b = 0; b < MB; ++b) a[b][h] = *(const i32x4_t*)(codes + b * 2048 + a_at[h]);
    }
    QRT_WAIT_LDS();  // the slot is in registers: the next step may overwrite it
    if (fetched < mine) {
      fetch(fetched, slot);
      ++fetched;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int b = 0; b < MB; ++b) acc[t][b] = IntProducts::add(w[t][h], a[b][h], acc[t][b]);
    slot = slot + 1 == U ? 0 : slot + 1;
  }
  __syncthreads();  // every wave has read its last slot: the rings' room now takes the sums
  int* red = (int*)rows_lds;  // [NW][NT][MB][4][64]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) red[(((wave * NT + t) * MB + b) * 4 + r) * 64 + lane] = acc[t][b][r];
  __syncthreads();
  // sum r of (tile, block, lane l): weight row 16 t + 4 (l / 16) + r, row 16 b + (l & 15)
  auto total = [&](int t, int b, int l, int r) {
    int s = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) s += red[(((w * NT + t) * MB + b) * 4 + r) * 64 + l];
    return (float)s;
  };
  constexpr int TILES_OUT = GATED && NT > 1 ? NT / 2 : NT;
  for (int i = threadIdx.x; i < TILES_OUT * MB * 256; i += 64 * NW) {
    const int l = i & 63, r = (i >> 6) & 3, b = (i >> 8) % MB, t = (i >> 8) / MB;
    const int m = 16 * b + (l & 15), in_tile = 4 * (l >> 4) + r;
    if (m >= p.M || (OUTS < 16 && in_tile >= OUTS)) continue;
    const int n = n0 + 16 * t + in_tile;
    if (n >= p.N) continue;
    const float sx = FUSED ? row_scale_of(most_of[m]) : p.a_scale[m];
    float y = total(t, b, l, r) * sx * p.w_scale[n];
    if constexpr (GATED) {
      const float u = total(NT > 1 ? t + NT / 2 : t, b, NT > 1 ? l : l + 32, r) * sx * p.w_scale[p.N + n];
      y = gated_act(y, u, p.ep.kind, p.ep.limit);
    }
    ((TO*)p.c)[(size_t)m * p.N + n] = from_f32<TO>(y);
  }
}

template <int NW, int WU, int MB, bool FEW, int U, bool GATED, int ROWS, int ITS, typename TX, typename TO>
static int launch_int8_rows(const Int8Rows& p, hipStream_t stream) {
  constexpr int NT = WU == 1 ? 1 : WU / 2, AU = FEW ? 1 : 2 * MB, OUTS = GATED ? 4 * WU : 8 * WU;
  constexpr size_t rings = (size_t)NW * U * (WU + (ITS ? 0 : AU)) * 1024, meet = (size_t)NW * NT * MB * 1024, most = 150 * 1024;
  const size_t smem = (rings > meet ? rings : meet) + (ITS ? (size_t)p.width * (4 * ROWS / fused_parts(p.M)) : 0);
  static_assert(rings <= most, "the rings of this configuration do not fit LDS");
  QRT_CHECK(smem <= most, "int8_rows: %d columns need %zu bytes of LDS", p.width, smem);
  auto kernel = int8_rows_kernel<NW, WU, MB, FEW, U, GATED, ROWS, ITS, TX, TO>;
  static bool allowed = false;  // once per kernel: not inside a stream capture again and again
  if (smem > 64 * 1024 && !allowed) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)most) != hipSuccess)
      return qrt_fail("int8_rows: cannot get %zu bytes of LDS", smem);
    allowed = true;
  }
  kernel<<<dim3((p.N + OUTS - 1) / OUTS), dim3(64 * NW), smem, stream>>>(p);
  QRT_LAUNCH_CHECK("int8_rows");
  return 0;
}

template <bool GATED, typename TX, typename TO>
static int fused_by_size(const Int8Rows& p, hipStream_t stream) {
  constexpr int WU = GATED ? 2 : 1;
  const int its = fused_its(p.M, p.width);
  if (p.M > 4) return launch_int8_rows<4, WU, 1, true, 4, GATED, 2, 2, TX, TO>(p, stream);
  if (its <= 2) return launch_int8_rows<4, WU, 1, true, 4, GATED, 1, 2, TX, TO>(p, stream);
  if (its <= 5) return launch_int8_rows<4, WU, 1, true, 4, GATED, 1, 5, TX, TO>(p, stream);
  return launch_int8_rows<4, WU, 1, true, 4, GATED, 1, FUSED_MOST, TX, TO>(p, stream);
}
template <bool GATED, typename TO>
static int rows_by_size(const Int8Rows& p, hipStream_t stream) {
  if constexpr (!GATED) {  // blocks are no more than compute units: eight waves each
    if (p.M <= 8 && p.N <= 4096) return launch_int8_rows<8, 2, 1, true, 4, false, 1, 0, float, TO>(p, stream);
    if (p.M <= 16 && p.N <= 4096) return launch_int8_rows<8, 2, 1, false, 4, false, 1, 0, float, TO>(p, stream);
    if (p.M <= 32 && p.N <= 4096) return launch_int8_rows<8, 2, 2, false, 3, false, 1, 0, float, TO>(p, stream);
  }
  if (p.M <= 8) return launch_int8_rows<4, 2, 1, true, 4, GATED, 1, 0, float, TO>(p, stream);
  if (p.M <= 16) return launch_int8_rows<4, 2, 1, false, 4, GATED, 1, 0, float, TO>(p, stream);
  // 32 weight rows a block fetch the activations half as often, where they leave as many blocks as compute units
  if (p.M <= 32) {
    if (p.N * (GATED ? 2 : 1) < 32 * 512) return launch_int8_rows<4, 2, 2, false, 3, GATED, 1, 0, float, TO>(p, stream);
    return launch_int8_rows<4, 4, 2, false, 2, GATED, 1, 0, float, TO>(p, stream);
  }
  if (p.N * (GATED ? 2 : 1) < 32 * 192) {
    if (p.M <= 48) return launch_int8_rows<4, 2, 3, false, 2, GATED, 1, 0, float, TO>(p, stream);
    return launch_int8_rows<4, 2, 4, false, 2, GATED, 1, 0, float, TO>(p, stream);
  }
  return launch_int8_rows<4, 4, 3, false, 2, GATED, 1, 0, float, TO>(p, stream);
}

// c [M, N] of up to 64 rows. Either x (rows as they are, in x_dtype: those that fused_takes, of a multiple of 8 columns) or a and a_scale.
// act_kind < 0: no gate; otherwise w is [2 N, width].
static int int8_rows(const void* x, int x_dtype, const void* a, const float* a_scale, const void* w, const float* w_scale, void* c, int out_dtype,
                     int M, int N, int K, int width, int act_kind, float limit, hipStream_t stream) {
  const Int8Rows p{x, (const int8_t*)a, a_scale, (const int8_t*)w, w_scale, c, M, N, K, width, GatedEpilogue{act_kind, limit, nullptr}};
  const bool bf = out_dtype == QRT_BF16;
#define GO(GATED)                                                                                                            \
  do {                                                                                                                       \
    if (x && x_dtype == QRT_BF16) return bf ? fused_by_size<GATED, bf16_t, bf16_t>(p, stream) : fused_by_size<GATED, bf16_t, float>(p, stream); \
    if (x) return bf ? fused_by_size<GATED, float, bf16_t>(p, stream) : fused_by_size<GATED, float, float>(p, stream);       \
    return bf ? rows_by_size<GATED, bf16_t>(p, stream) : rows_by_size<GATED, float>(p, stream);                              \
  } while (0)
  if (act_kind >= 0) GO(true);
  GO(false);
#undef GO
}

// Whether the weight is streamed past the rows; more go by tiles. us by streams and tiles at 48 and 64 rows: 6,144 x 4,096 12.5, 14.0 and 14.0, 14.0; gated
// 9,728 x 2,560 19.7, 25.4 and 21.2, 21.2; 2,560 x 9,728 19.9, 23.0 and 26.3, 26.3.
constexpr bool streams(int M, int N, bool gated) { return M <= 48 || (M <= 64 && N * (gated ? 2 : 1) < 32 * 192); }

static int64_t codes_room(int M, int width) { return (int64_t)M * width + 4 * (((int64_t)M + 3) & ~3ll); }

// Bytes of workspace that qrt_int8_product wants: none, or the rows' codes and scales; always these with parts of K.
extern "C" int64_t qrt_int8_workspace(int M, int N, int K, int width) {
  return K % 8 == 0 && fused_takes(M, N, width) ? 0 : codes_room(M, width);
}

static int int8_product(const void* x, int x_dtype, const float* codes_scale, const void* w, const float* w_scale, void* c, int out_dtype, void* workspace, int M, int N,
                        int K, int width, int tile, int parts, int act_kind, float limit, hipStream_t stream) {
  if (check_width("int8_product", M, K, width)) return -1;
  QRT_CHECK(N > 0 && N < (1 << 30), "int8_product: bad size N=%d", N);
  QRT_CHECK(x_dtype == QRT_BF16 || x_dtype == QRT_F32, "int8_product: unknown dtype %d", x_dtype);
  QRT_CHECK(out_dtype == QRT_BF16 || out_dtype == QRT_F32, "int8_product: unknown output dtype %d", out_dtype);
  QRT_CHECK(act_kind <= QRT_ACT_CLAMPED, "int8_product: unknown activation %d", act_kind);
  QRT_CHECK(((uintptr_t)w | (uintptr_t)c | (uintptr_t)workspace) % 16 == 0, "int8_product: operands must begin at multiples of 16 bytes");
  if (codes_scale) {
    QRT_CHECK((uintptr_t)x % 16 == 0, "int8_product: codes must begin at a multiple of 16 bytes");
    if (M == 0) return 0;
    if (parts == 1 && streams(M, N, act_kind >= 0)) return int8_rows(nullptr, x_dtype, x, codes_scale, w, w_scale, c, out_dtype, M, N, K, width, act_kind, limit, stream);
    return int8_tiles(x, codes_scale, w, w_scale, c, out_dtype, M, N, width, tile, parts, act_kind, limit, stream);
  }
  const int64_t room = parts == 1 ? qrt_int8_workspace(M, N, K, width) : codes_room(M, width);
  QRT_CHECK(room == 0 || workspace, "int8_product: %d rows of %d columns need a workspace", M, K);
  QRT_CHECK(room > 0 || (uintptr_t)x % 16 == 0, "int8_product: rows must begin at a multiple of 16 bytes");
  if (M == 0) return 0;
  if (room == 0) return int8_rows(x, x_dtype, nullptr, nullptr, w, w_scale, c, out_dtype, M, N, K, width, act_kind, limit, stream);
  int8_t* const codes = (int8_t*)workspace;
  float* const scale = (float*)(codes + (int64_t)M * width);
  if (qrt_quantize_rows(x, x_dtype, codes, scale, M, K, width, stream)) return -1;
  if (parts == 1 && streams(M, N, act_kind >= 0)) return int8_rows(nullptr, x_dtype, codes, scale, w, w_scale, c, out_dtype, M, N, K, width, act_kind, limit, stream);
  return int8_tiles(codes, scale, w, w_scale, c, out_dtype, M, N, width, tile, parts, act_kind, limit, stream);
}

// c [M, N] (out_dtype) = rows x [M, K] (x_dtype) by w [N, width] and w_scale [N], or with a gate (act_kind >= 0) w [2 N, width], w_scale [2 N] and the activation
// of the two. With codes_scale [M] (not null) x is codes already, [M, width]. tile: a number of TILES in ops/hip.py, for more than 48 rows.
extern "C" int qrt_int8_product(const void* x, int x_dtype, const float* codes_scale, const void* w, const float* w_scale, void* c, int out_dtype, void* workspace, int M, int N,
                                int K, int width, int tile, int act_kind, float limit, hipStream_t stream) {
  return int8_product(x, x_dtype, codes_scale, w, w_scale, c, out_dtype, workspace, M, N, K, width, tile, 1, act_kind, limit, stream);
}
// The same without a gate, by tiles whatever M: planes c [parts, M, N] in float32 whose sum is the product, two parts of K or more.
extern "C" int qrt_int8_planes(const void* x, int x_dtype, const float* codes_scale, const void* w, const float* w_scale, void* c, void* workspace, int M, int N, int K, int width,
                               int tile, int parts, hipStream_t stream) {
  QRT_CHECK(parts > 1, "int8_planes: %d parts of K", parts);
  return int8_product(x, x_dtype, codes_scale, w, w_scale, c, QRT_F32, workspace, M, N, K, width, tile, parts, -1, 0.f, stream);
}
