// Products of many rows of 8-bit integers by tiles through LDS: tiles.h has the loop, whose stages of 128 bytes are 128 columns
// here, and the sums are whole numbers. The scales of rows and channels multiply at the end, then the gate if there is one.
// int8_rows has what is computed; everything behind the sums is as in the tiles of bfloat16, and so is the choice of the tile: bytes and
// cycles of a stage are the same (the best of all tiles was within 2 % of the one chosen).
// The matrix cores bound it. us and 10^15 operations a second, without the rows' codes: 2,048 rows by 2,560 x 9,728 48.7, 2.1; gated, 1,999 rows by
// 2 x 9,728 x 2,560 107, 1.86 (the gate's epilogue); 8,192 by 8,192 x 8,192 509, 2.16, where the vendor's library takes 493, and 73.8 and 115 for
// the first two, without scales and gate. Tiles of 32 x 32 x 32 products were slower: 55 and 119 us.
#include "common.h"
#include "direct.h"
#include "gemm_epilogue.h"
#include "int8.h"
#include "tiles.h"

struct Int8TileArgs {
  const int8_t* A;
  const float* a_scale;
  const int8_t* W;
  const float* w_scale;
  void* C;
  int M, N, width;
  int mtiles, ntiles;
  int parts;  // of K, a plane [M, N] each
  int kind;
  float limit;
};

template <int BM, int BN, int WN, bool GATED, typename TO>
constexpr int int8_result_bytes() {
  return sizeof(TO) == 4 ? 0 : BM * ((GATED ? BN : 2 * BN) + 16 * WN);
}
template <int BM, int BN, int WM, int WN, int S, bool GATED, typename TO>
constexpr size_t int8_tile_lds() {
  typedef Tile<BM, BN, WM, WN, S, IntProducts> T;
  constexpr size_t result = int8_result_bytes<BM, BN, WN, GATED, TO>(), both = result + T::STAGE;
  constexpr size_t least = T::RING > result ? T::RING : result;
  static_assert(least <= 160 * 1024, "the result of this tile does not fit LDS");
  return result > 0 && both > least && both <= 160 * 1024 ? both : least;
}

template <int BM, int BN, int WM, int WN, int S, bool GATED, typename TO>
__global__ __launch_bounds__(64 * WM * WN, 2) void int8_tiles_kernel(Int8TileArgs p) {
#ifdef __HIP_DEVICE_COMPILE__  // the host's compiler knows no buffer resources
  typedef Tile<BM, BN, WM, WN, S, IntProducts> T;
  constexpr int TM = T::TM, TN = T::TN;
  extern __shared__ __align__(16) unsigned char tiles_lds[];  // [S] stages, then the result
  const int lane = threadIdx.x & 63, wave = uniform_wave_number();
  const int wm = wave / WN, wn = wave % WN;
  const int r16 = lane & 15, quad = lane >> 4;

  // Blocks reach the XCDs in turn: each gets a run of neighbouring tiles, down bands of some 2,048 rows, column by column.
  const int total = p.mtiles * p.ntiles * p.parts;
  int m0, n0, part, s0, stages;
  unsigned aoff[T::AL], woff[T::WL];  // rows past the end repeat the last one and are not stored
  auto locate = [&](int tile) {
    const int xcd = tile & 7;
    int id = xcd * (total >> 3) + min(xcd, total & 7) + (tile >> 3);
    part = id / (p.mtiles * p.ntiles);
    id -= part * p.mtiles * p.ntiles;
    constexpr int BAND = 2048 / BM;
    const int band = id / (BAND * p.ntiles), in_band = id - band * BAND * p.ntiles;
    const int high = min(BAND, p.mtiles - band * BAND);
    m0 = (band * BAND + in_band % high) * BM;
    n0 = in_band / high * (GATED ? BN / 2 : BN);
    const int all = p.width / INT8_STAGE, each = (all + p.parts - 1) / p.parts;
    s0 = min(all, part * each);
    stages = min(all, s0 + each) - s0;
#pragma unroll
    for (int j = 0; j < T::AL; ++j)
      aoff[j] = (unsigned)min(m0 + T::row_of(j, T::AU, wave, lane), p.M - 1) * (unsigned)p.width + T::piece_of(lane);
#pragma unroll
    for (int j = 0; j < T::WL; ++j) {
      const int in_tile = T::row_of(j, T::WU, wave, lane);
      const int row = GATED ? min(n0 + 8 * (in_tile >> 4) + (in_tile & 7), p.N - 1) + ((in_tile & 8) ? p.N : 0)
                            : min(n0 + in_tile, p.N - 1);
      woff[j] = (unsigned)row * (unsigned)p.width + T::piece_of(lane);
    }
  };
  const __amdgpu_buffer_rsrc_t a_buf = T::buffer(p.A, (size_t)p.M * p.width);
  const __amdgpu_buffer_rsrc_t w_buf = T::buffer(p.W, (size_t)(GATED ? 2 : 1) * p.N * p.width);

  constexpr int RESULT = int8_result_bytes<BM, BN, WN, GATED, TO>();
  constexpr int FIRST = RESULT == 0 ? S : ((int)int8_tile_lds<BM, BN, WM, WN, S, GATED, TO>() - RESULT) / T::STAGE;
  unsigned char* const result = tiles_lds + int8_tile_lds<BM, BN, WM, WN, S, GATED, TO>() - RESULT;
  int tile = blockIdx.x, fetched = 0;
  locate(tile);
  while (true) {
    i32x4_t acc[TM][TN];
    T::template products<0>(a_buf, w_buf, aoff, woff, s0, stages, tiles_lds, fetched, acc);
    QRT_WAIT_LDS();
    QRT_BARRIER();  // nobody reads the ring any more
    // acc[i][j][r]: row 16 i + r16 of the wave's result, row 16 j + 4 quad + r of its weights
    constexpr int ROWS = BM / WM, COLS = (GATED ? 8 : 16) * TN;
    const int mw = m0 + wm * ROWS, nw = n0 + wn * COLS;
    // the scales come in front of the next tile's loads, so that they are not waited for behind them
    float sx[TM], sw[TN][4];
#pragma unroll
    for (int i = 0; i < TM; ++i) sx[i] = p.a_scale[min(mw + 16 * i + r16, p.M - 1)];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        sw[j][r] = p.w_scale[GATED ? min(nw + 8 * j + 4 * (quad & 1) + r, p.N - 1) + (quad & 2 ? p.N : 0) : min(nw + 16 * j + 4 * quad + r, p.N - 1)];
    TO* C = (TO*)p.C + (size_t)part * p.M * p.N;
    const bool more = tile + (int)gridDim.x < total;
    tile += gridDim.x;
    if (more) {
      locate(tile);
      T::template fetch_first<0>(a_buf, w_buf, aoff, woff, s0, stages, tiles_lds, 0, FIRST);
    }
    constexpr int PITCH = 2 * COLS + 16;
    unsigned char* own = result + wave * ROWS * PITCH;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = mw + 16 * i + r16;
      unsigned char* row = own + (16 * i + r16) * PITCH;
      // GATED: the lower half of the lanes holds gate values and the upper half the up values that belong to them: two
      // tiles change halves, and every lane has a gate and an up value; a last single tile leaves the upper half idle
#pragma unroll
      for (int j = 0; j < TN; j += GATED ? 2 : 1) {
        float o[4];
        bool any = true;
        int in_row;
        if constexpr (GATED) {
          const int j2 = j + 1 < TN ? j + 1 : j;
          float g[4], u[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            g[r] = (float)acc[i][j][r] * sx[i] * sw[j][r], u[r] = (float)acc[i][j2][r] * sx[i] * sw[j2][r];
            swap_halves(g[r], u[r]);
          }
          if constexpr (sizeof(TO) == 2) gated_act4(g, u, p.kind, p.limit, o);
          else
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = gated_act(g[r], u[r], p.kind, p.limit);
          any = j + 1 < TN || quad < 2;
          in_row = 8 * (j + (quad >> 1)) + 4 * (quad & 1);
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = (float)acc[i][j][r] * sx[i] * sw[j][r];
          in_row = 16 * j + 4 * quad;
        }
        if constexpr (sizeof(TO) == 2) {
          if (any) store4((bf16_t*)(row + 2 * in_row), o);
        } else if (any && m < p.M) {
          const int n = nw + in_row;
          float* to = C + (size_t)m * p.N + n;
          if (p.N % 4 == 0) {
            if (n < p.N) store4(to, o);
          } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (n + r < p.N) to[r] = o[r];
          }
        }
      }
    }
    if constexpr (sizeof(TO) == 2) {
      constexpr int PIECES = COLS / 8;  // of 16 bytes in a row
#pragma unroll
      for (int c0 = 0; c0 < ROWS * PIECES; c0 += 64) {
        const int c = c0 + lane, row = c / PIECES, at = c % PIECES;
        if (ROWS * PIECES % 64 && c >= ROWS * PIECES) break;
        const u32x4_t v = *(const u32x4_t*)(own + row * PITCH + 16 * at);
        const int m = mw + row, n = nw + 8 * at;
        if (m >= p.M) continue;
        if (p.N % 8 == 0) {
          if (n < p.N) *(u32x4_t*)(C + (size_t)m * p.N + n) = v;
        } else {
          const bf16x8_t e = __builtin_bit_cast(bf16x8_t, v);
#pragma unroll
          for (int r = 0; r < 8; ++r)
            if (n + r < p.N) C[(size_t)m * p.N + n + r] = e[r];
        }
      }
    }
    if (!more) break;
    fetched = FIRST < S ? FIRST : S;
    QRT_WAIT_LDS();
    QRT_BARRIER();  // the result's room is the ring's again
  }
#endif
}

template <int BM, int BN, int WM, int WN, int S, bool GATED, typename TO>
static int launch_int8_tiles(Int8TileArgs p, hipStream_t stream) {
  constexpr size_t smem = int8_tile_lds<BM, BN, WM, WN, S, GATED, TO>();
  const int outs = GATED ? BN / 2 : BN;
  p.mtiles = (p.M + BM - 1) / BM;
  p.ntiles = (p.N + outs - 1) / outs;
  const int64_t blocks = (int64_t)p.mtiles * p.ntiles * p.parts;
  QRT_CHECK(blocks < (1 << 30), "int8_tiles: too many tiles for one launch (M=%d N=%d)", p.M, p.N);
  auto kernel = int8_tiles_kernel<BM, BN, WM, WN, S, GATED, TO>;
  static bool allowed = false;  // once per kernel: not inside a stream capture again and again
  if (smem > 64 * 1024 && !allowed) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != hipSuccess)
      return qrt_fail("int8_tiles: cannot get %zu bytes of LDS", smem);
    allowed = true;
  }
  constexpr int64_t resident = 256 * (160 * 1024 / smem);  // blocks that the compute units hold
  kernel<<<(unsigned)(blocks < resident ? blocks : resident), 64 * WM * WN, smem, stream>>>(p);
  QRT_LAUNCH_CHECK("int8_tiles");
  return 0;
}

template <int BM, int BN, int WM, int WN, int S>
static int int8_by_result(const Int8TileArgs& p, int out_dtype, hipStream_t stream) {
  if (p.kind >= 0) {
    if (out_dtype == QRT_F32) return launch_int8_tiles<BM, BN, WM, WN, S, true, float>(p, stream);
    return launch_int8_tiles<BM, BN, WM, WN, S, true, bf16_t>(p, stream);
  }
  if (out_dtype == QRT_F32) return launch_int8_tiles<BM, BN, WM, WN, S, false, float>(p, stream);
  return launch_int8_tiles<BM, BN, WM, WN, S, false, bf16_t>(p, stream);
}

// c [M, N] from codes a [M, width], w [N, width] ([2 N, width] with a gate: act_kind >= 0), or with parts > 1 (no gate, float32) planes [parts, M, N];
// tile: a number of TILES in ops/hip.py.
int int8_tiles(const void* a, const float* a_scale, const void* w, const float* w_scale, void* c, int out_dtype, int M, int N, int width, int tile,
               int parts, int act_kind, float limit, hipStream_t stream) {
  const uint64_t limit_bytes = (1ull << 32) - 128;  // offsets are 32 bits
  QRT_CHECK((uint64_t)M * width <= limit_bytes && (uint64_t)(act_kind >= 0 ? 2 : 1) * N * width <= limit_bytes,
            "int8_tiles: an operand of 4 GiB or more (M=%d N=%d, rows of %d)", M, N, width);
  QRT_CHECK(parts == 1 || (parts > 1 && parts <= 64 && act_kind < 0 && out_dtype == QRT_F32), "int8_tiles: %d parts of K need no gate and float32 output", parts);
  const int stages = width / INT8_STAGE, each = (stages + parts - 1) / parts;
  QRT_CHECK(each * (parts - 1) < stages, "int8_tiles: %d parts of %d stages leave one without any", parts, stages);
  const Int8TileArgs p{(const int8_t*)a, a_scale, (const int8_t*)w, w_scale, c, M, N, width, 0, 0, parts, act_kind, limit};
  switch (tile) {
    case 0: return int8_by_result<256, 192, 4, 2, 2>(p, out_dtype, stream);
    case 1: return int8_by_result<256, 160, 4, 2, 3>(p, out_dtype, stream);
    case 2: return int8_by_result<256, 128, 4, 2, 3>(p, out_dtype, stream);
    case 3: return int8_by_result<192, 192, 4, 2, 3>(p, out_dtype, stream);
    case 4: return int8_by_result<192, 160, 4, 2, 3>(p, out_dtype, stream);
    case 5: return int8_by_result<192, 128, 4, 2, 3>(p, out_dtype, stream);
    case 6: return int8_by_result<128, 160, 2, 2, 4>(p, out_dtype, stream);
    case 7: return int8_by_result<128, 128, 2, 2, 4>(p, out_dtype, stream);
    case 8: return int8_by_result<128, 96, 2, 2, 4>(p, out_dtype, stream);
    case 9: return int8_by_result<96, 160, 2, 2, 4>(p, out_dtype, stream);
    case 10: return int8_by_result<96, 96, 2, 2, 6>(p, out_dtype, stream);
    case 11: return int8_by_result<128, 64, 2, 2, 6>(p, out_dtype, stream);
    case 12: return int8_by_result<64, 64, 1, 4, 4>(p, out_dtype, stream);
    case 13: return int8_by_result<64, 128, 1, 4, 3>(p, out_dtype, stream);
    default: return qrt_fail("int8_tiles: no tile %d", tile);
  }
}
