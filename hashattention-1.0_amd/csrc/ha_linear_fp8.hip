// y = x W^T with x and W in e4m3, one fp32 scale per block of 128 inputs of a row of x and per 128 x 128 block of W:
//
//   out[m, n] = sum_kb xs[m, kb] * ws[n, kb] * sum_{k in block kb} xq[m, k] * wq[n, k]
//
// The inner sum runs on the matrix cores, the outer one is an fp32 FMA per output and block.
//
// Which matrix instruction.  The 8-bit ones (v_mfma_f32_16x16x128_f8f6f4, v_mfma_f32_16x16x32_fp8_fp8) add eight neighbouring
// products at a time and drop what lies more than 13 bits below the largest of the eight (measured: 2^3 beside 2^16 is kept,
// 2^2 is lost, wherever the two sit within eight inputs; further apart the sum is fp32).  On normally distributed numbers that
// is 1.5e-5 of the result, 1e-4 where magnitudes spread widely.  e4m3 numbers are exact in bf16 and v_mfma_f32_16x16x32_bf16
// keeps its sums in fp32 (1.2e-8 on the same numbers), at half the 8-bit rate plus one conversion per two numbers.
//
//   ha_weight_fp8_bytes / ha_weight_fp8_scales / ha_pack_weight_fp8   the packed weights
//   ha_linear_fp8                                                     the product, residual or SwiGLU behind
#include "ha_fp8.h"

namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTileRows = 16;
constexpr int kTileBytes = kTileRows * HA_FP8_BLOCK;  // 2 KiB

// Packed weights.  Tile (nt, kb) holds 16 rows x 128 inputs as two pieces of one KiB; lane l of a wave reads its 16 bytes of each
// piece at l * 16 - row l % 16, inputs 64 p + 16 (l / 16) .. + 15 of piece p - and has the A operand of the matrix instruction.
// (x is read in the same order, so which input of the block sits in which byte does not matter to the sum.)  Rows and inputs
// beyond the matrix are zero.  `glu`: the matrix is [F gate rows; F up rows] and tile nt holds gate rows 8 nt .. 8 nt + 7 and then
// the up rows of the same columns: a tile's 16 sums are 8 activated outputs.
// Scales: two numbers per tile, rows 0 - 7 and rows 8 - 15 (gate and up have blocks of their own).
struct Packed {
    int n_tiles, kb;
};
static inline Packed packed_shape(int N, int K, int glu) {
    const int rows = glu ? N / 2 : N, per = glu ? 8 : kTileRows;
    return {rows / per + (rows % per != 0), ha_fp8_blocks(K)};
}

__device__ __forceinline__ float fp8_to_float(uint32_t byte) { return __builtin_amdgcn_cvt_f32_fp8((int)byte, 0); }

// One workgroup per block of 128 rows x 128 inputs of one matrix (blockIdx.y: row block; glu: those of gate, then those of up):
// its largest magnitude and its scale (or the scale given), then the block's 1024 pieces of 16 bytes, four per thread.
// dtype HA_FP8_E4M3: the numbers are taken over as they are.
__global__ __launch_bounds__(256) void pack_fp8_kernel(const void *__restrict__ w, int64_t w_sn, int dtype, const float *__restrict__ given,
                                                       int64_t given_sn, int rows, int row_blocks, int K, int kb_count, int glu,
                                                       int n_tiles, uint8_t *__restrict__ tiles, float *__restrict__ scales) {
    __shared__ uint32_t s_top[4];
    const int tid = threadIdx.x, kb = blockIdx.x, half = (int)blockIdx.y / row_blocks, nb = (int)blockIdx.y % row_blocks;
    float v[4][16];
    uint32_t top = 0u;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int r = nb * 128 + (tid >> 3) + 32 * p, k0 = kb * 128 + (tid & 7) * 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float f = 0.f;
            if (r < rows && k0 + i < K) {
                const int64_t at = ((int64_t)half * rows + r) * w_sn + k0 + i;
                f = dtype == HA_FP8_E4M3 ? fp8_to_float(((const uint8_t *)w)[at]) : ha_load_elem(w, at, dtype);
            }
            v[p][i] = f;
            top = max(top, ha_abs_bits(f));
        }
    }
    HaFp8Scale s = {1.0f, 1.0f};
    if (dtype == HA_FP8_E4M3) {
        s.scale = given[(int64_t)blockIdx.y * given_sn + kb];
    } else {
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        if ((tid & 63) == 0) s_top[tid >> 6] = top;
        __syncthreads();
        s = ha_fp8_scale(max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3])));
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int r = nb * 128 + (tid >> 3) + 32 * p, piece = tid & 7;
        const int nt = glu ? r >> 3 : r >> 4, tr = glu ? (half << 3) | (r & 7) : r & 15;
        if (nt >= n_tiles) continue;
        const int64_t tile = (int64_t)nt * kb_count + kb;
        uint4 b;
        b.x = ha_fp8x4(v[p][0] * s.inv, v[p][1] * s.inv, v[p][2] * s.inv, v[p][3] * s.inv);
        b.y = ha_fp8x4(v[p][4] * s.inv, v[p][5] * s.inv, v[p][6] * s.inv, v[p][7] * s.inv);
        b.z = ha_fp8x4(v[p][8] * s.inv, v[p][9] * s.inv, v[p][10] * s.inv, v[p][11] * s.inv);
        b.w = ha_fp8x4(v[p][12] * s.inv, v[p][13] * s.inv, v[p][14] * s.inv, v[p][15] * s.inv);
        // piece of 16 inputs number `piece` of the block: KiB piece / 4, lane group piece % 4
        *reinterpret_cast<uint4 *>(tiles + tile * kTileBytes + (piece >> 2) * 1024 + ((piece & 3) * 16 + tr) * 16) = b;
        if (piece == 0) {
            if (glu) {
                if ((r & 7) == 0) scales[tile * 2 + half] = s.scale;
            } else if ((r & 7) == 0) {
                scales[tile * 2 + ((r >> 3) & 1)] = s.scale;
            }
        }
    }
}

// eight e4m3 numbers as bf16, exactly: a lane's share of the operand of v_mfma_f32_16x16x32_bf16
__device__ __forceinline__ bf16x8 widen8(uint32_t lo, uint32_t hi) {
    const i32x4 v = {__builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, false)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)lo, 1.0f, true)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, false)),
                     __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)hi, 1.0f, true))};
    return __builtin_bit_cast(bf16x8, v);
}
// a lane's 32 numbers of a block of 128 inputs (its two pieces)
struct Wide {
    bf16x8 v[4];
};
__device__ __forceinline__ Wide widen(const uint4 &a, const uint4 &b) {
    return {{widen8(a.x, a.y), widen8(a.z, a.w), widen8(b.x, b.y), widen8(b.z, b.w)}};
}
__device__ __forceinline__ f32x4 block_sum(const Wide &w, const Wide &x) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], c, 0, 0, 0);
    return c;
}

struct Epilogue {
    const void *res;
    int64_t res_sm;
    void *out;
    int64_t out_sm;
    int out_dtype;
};

// The simple form, for any size: one tile of 16 weight rows and 16 MT rows of x per workgroup, the blocks of K dealt out to its
// waves, their sums joined through LDS.
template <int NWAVE, int MT, bool GLU>
__global__ __launch_bounds__(NWAVE * 64) void linear_fp8_kernel(const uint8_t *__restrict__ x, int64_t x_sm, const float *__restrict__ xs,
                                                                int64_t xs_sm, const uint8_t *__restrict__ tiles,
                                                                const float *__restrict__ ws, Epilogue ep, int M, int N, int kb_count,
                                                                int n_tiles) {
    __shared__ float s_c[NWAVE][16][16 * MT + 1];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int nt = (int)(blockIdx.x % (unsigned)n_tiles), m0 = (int)(blockIdx.x / (unsigned)n_tiles) * 16 * MT;
    const uint8_t *tp = tiles + (int64_t)nt * kb_count * kTileBytes + lane * 16;
    const float *wsp = ws + (int64_t)nt * kb_count * 2 + (g >> 1);
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int kb = wave; kb < kb_count; kb += NWAVE) {
        const uint4 *wt = reinterpret_cast<const uint4 *>(tp + (int64_t)kb * kTileBytes);
        const Wide wv = widen(wt[0], wt[64]);
        const float w_scale = wsp[2 * kb];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int m = m0 + 16 * t + r;
            uint4 a = make_uint4(0u, 0u, 0u, 0u), b = a;
            float s = 0.f;
            if (m < M) {
                const uint4 *xp = reinterpret_cast<const uint4 *>(x + m * x_sm + kb * HA_FP8_BLOCK + g * 16);
                a = xp[0];
                b = xp[4];
                s = xs[m * xs_sm + kb] * w_scale;
            }
            const f32x4 part = block_sum(wv, widen(a, b));
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(part[i], s, acc[t][i]);
        }
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_c[wave][4 * g + i][16 * t + r] = acc[t][i];
    __syncthreads();
    auto total = [&](int row, int mm) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < NWAVE; ++w) y += s_c[w][row][mm];
        return y;
    };
    if constexpr (GLU) {
        for (int t = tid; t < 8 * 16 * MT; t += NWAVE * 64) {
            const int mm = t >> 3, c = t & 7, col = 8 * nt + c;
            if (m0 + mm >= M || col >= N / 2) continue;
            const float gate = total(c, mm);
            ha_store_elem(ep.out, (m0 + mm) * ep.out_sm + col, gate / (1.0f + expf(-gate)) * total(8 + c, mm), ep.out_dtype);
        }
    } else {
        for (int t = tid; t < 16 * 16 * MT; t += NWAVE * 64) {
            const int mm = t >> 4, c = t & 15, n = 16 * nt + c;
            if (m0 + mm >= M || n >= N) continue;
            float y = total(c, mm);
            if (ep.res) y += ha_load_elem(ep.res, (m0 + mm) * ep.res_sm + n, ep.out_dtype);
            ha_store_elem(ep.out, (m0 + mm) * ep.out_sm + n, y, ep.out_dtype);
        }
    }
}

}  // namespace

extern "C" {

int64_t ha_weight_fp8_bytes(int N, int K, int glu) {
    if (N < 1 || K < 1 || (glu && N % 2 != 0)) return 0;
    const Packed p = packed_shape(N, K, glu);
    return (int64_t)p.n_tiles * p.kb * kTileBytes;
}

int64_t ha_weight_fp8_scales(int N, int K, int glu) { return ha_weight_fp8_bytes(N, K, glu) / kTileBytes * 2; }

int ha_pack_weight_fp8(const void *w, int64_t w_stride_n, int dtype, const float *w_scales, int64_t w_scales_stride_n, int N, int K, int glu,
                       void *tiles, float *tile_scales, void *stream) {
    HA_REQUIRE(w && tiles && tile_scales, HA_ERR_NULL_POINTER, "w/tiles/tile_scales is NULL");
    HA_REQUIRE(dtype == HA_F32 || dtype == HA_BF16 || dtype == HA_F16 || dtype == HA_FP8_E4M3, HA_ERR_BAD_DTYPE, "unknown dtype %d", dtype);
    HA_REQUIRE((dtype == HA_FP8_E4M3) == (w_scales != nullptr), HA_ERR_NULL_POINTER,
               "weights in e4m3 come with their scales, any other type without");
    HA_REQUIRE(N >= 1 && K >= 1 && w_stride_n >= K && (glu == 0 || (glu == 1 && N % 2 == 0)), HA_ERR_BAD_SHAPE,
               "need N, K >= 1, an even N for the gate/up form, rows of at least K elements");
    const Packed p = packed_shape(N, K, glu);
    const int rows = glu ? N / 2 : N, row_blocks = ha_fp8_blocks(rows);
    HA_REQUIRE(!w_scales || w_scales_stride_n >= p.kb, HA_ERR_BAD_SHAPE, "a row of w_scales holds a number for every block of 128 inputs");
    HA_REQUIRE(row_blocks * (glu ? 2LL : 1LL) <= 65535, HA_ERR_BAD_SHAPE, "matrix too large for one launch");
    HA_REQUIRE(ha_aligned(w, dtype == HA_FP8_E4M3 ? 1 : ha_dtype_bytes(dtype)) && ha_aligned(w_scales, 4) && ha_aligned(tiles, 16) &&
                   ha_aligned(tile_scales, 8),
               HA_ERR_MISALIGNED, "tiles must be 16-byte aligned, the others to their elements");
    int st = ha_require_device();
    if (st) return st;
    hipLaunchKernelGGL(pack_fp8_kernel, dim3((unsigned)p.kb, (unsigned)(row_blocks * (glu ? 2 : 1))), dim3(256), 0, (hipStream_t)stream, w,
                       w_stride_n, dtype, w_scales, w_scales_stride_n, rows, row_blocks, K, p.kb, glu, p.n_tiles, (uint8_t *)tiles, tile_scales);
    HA_CHECK_LAUNCH("pack_fp8_kernel");
    return HA_OK;
}

int ha_linear_fp8(const void *xq, int64_t xq_stride_m, const float *x_scales, int64_t x_scales_stride_m, const void *tiles,
                  const float *tile_scales, const void *residual, int64_t residual_stride_m, int act, void *out, int64_t out_stride_m,
                  int out_dtype, int M, int N, int K, void *stream) {
    HA_REQUIRE(tiles && tile_scales && (M == 0 || (xq && x_scales && out)), HA_ERR_NULL_POINTER,
               "xq/x_scales/tiles/tile_scales/out is NULL");
    HA_REQUIRE(out_dtype == HA_F32 || out_dtype == HA_BF16 || out_dtype == HA_F16, HA_ERR_BAD_DTYPE, "unknown dtype %d", out_dtype);
    HA_REQUIRE(M >= 0 && N >= 1 && K >= 1, HA_ERR_BAD_SHAPE, "need M >= 0, N >= 1, K >= 1");
    HA_REQUIRE(act == HA_ACT_NONE || act == HA_ACT_SWIGLU, HA_ERR_BAD_SHAPE, "unknown activation %d", act);
    HA_REQUIRE(!act || (N % 2 == 0 && !residual), HA_ERR_BAD_SHAPE, "SwiGLU needs an even number of weight rows and no residual");
    const Packed p = packed_shape(N, K, act);
    const int n_out = act ? N / 2 : N;
    HA_REQUIRE(xq_stride_m >= (int64_t)p.kb * HA_FP8_BLOCK && x_scales_stride_m >= p.kb && out_stride_m >= n_out &&
                   (!residual || residual_stride_m >= N),
               HA_ERR_BAD_SHAPE, "strides smaller than the rows they span");
    const int es = ha_dtype_bytes(out_dtype);
    HA_REQUIRE(ha_aligned(xq, 16) && xq_stride_m % 16 == 0 && ha_aligned(tiles, 16), HA_ERR_MISALIGNED,
               "rows of xq and tiles must be 16-byte aligned");
    HA_REQUIRE(ha_aligned(x_scales, 4) && ha_aligned(tile_scales, 8) && ha_aligned(out, es) && ha_aligned(residual, es), HA_ERR_MISALIGNED,
               "pointers are not aligned to their elements");
    int st = ha_require_device();
    if (st || M == 0) return st;
    const Epilogue ep = {residual, residual_stride_m, out, out_stride_m, out_dtype};
    const int MT = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const int64_t grid = (int64_t)p.n_tiles * ((M + 16LL * MT - 1) / (16 * MT));
    HA_REQUIRE(grid <= 2147483647LL, HA_ERR_BAD_SHAPE, "too many tiles for one launch");
#define HA_LINEAR(NW_, MT_, G_)                                                                                                          \
    hipLaunchKernelGGL((linear_fp8_kernel<NW_, MT_, G_>), dim3((unsigned)grid), dim3(NW_ * 64), 0, (hipStream_t)stream, (const uint8_t *)xq, \
                       xq_stride_m, x_scales, x_scales_stride_m, (const uint8_t *)tiles, tile_scales, ep, M, N, p.kb, p.n_tiles)
    if (MT == 1) {
        if (act) HA_LINEAR(8, 1, true);
        else HA_LINEAR(8, 1, false);
    } else if (MT == 2) {
        if (act) HA_LINEAR(8, 2, true);
        else HA_LINEAR(8, 2, false);
    } else {
        if (act) HA_LINEAR(8, 4, true);
        else HA_LINEAR(8, 4, false);
    }
#undef HA_LINEAR
    HA_CHECK_LAUNCH("linear_fp8_kernel");
    return HA_OK;
}

}  // extern "C"
