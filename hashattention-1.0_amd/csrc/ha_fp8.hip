// Rows in 8 bits with a scale per block of 128, written by the operators that stand in front of the 8-bit projections:
//
//   ha_quantize_rows_fp8   rows as they are (the attention output in front of its projection)
//   ha_rmsnorm_fp8         the residual's addition and the root-mean-square norm (in front of QKV and of gate/up)
//   ha_swiglu_fp8          silu(gate) * up (in front of the down projection)
//
// Each is one pass: the elements are read once, stay in registers in fp32 and are rounded once, to 8 bits.
#include "ha_fp8.h"

namespace {

template <typename E>
constexpr int dtype_of = __is_same(E, ElemF32) ? HA_F32 : __is_same(E, ElemBF16) ? HA_BF16 : HA_F16;

// Rows begin anywhere (an odd width moves every row off the last one's alignment): 16 bytes at the address of an element are one
// load all the same, which the hardware takes at any alignment.
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_anywhere __attribute__((aligned(2)));
template <typename E>
struct Eight {
    u32x4 v[Elem<E>::bytes / 2];
};

// eight consecutive elements row[k0 .. k0 + 8) of a row of K, zero beyond K
template <typename E>
__device__ __forceinline__ Eight<E> load8(const char *row, int k0, int K) {
    constexpr int es = Elem<E>::bytes;
    Eight<E> r;
    if (k0 + 8 <= K) {
        const u32x4_anywhere *p = reinterpret_cast<const u32x4_anywhere *>(row + (int64_t)k0 * es);
#pragma unroll
        for (int i = 0; i < es / 2; ++i) r.v[i] = p[i];
        return r;
    }
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = k0 + i >= K ? 0u : es == 4 ? ((const uint32_t *)row)[k0 + i] : (uint32_t)((const uint16_t *)row)[k0 + i];
    if constexpr (es == 4) {
        r.v[0] = u32x4{w[0], w[1], w[2], w[3]};
        r.v[1] = u32x4{w[4], w[5], w[6], w[7]};
    } else {
        r.v[0] = u32x4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
    }
    return r;
}
template <typename E>
__device__ __forceinline__ void to_float(const Eight<E> &r, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if constexpr (Elem<E>::bytes == 4)
            f[i] = __uint_as_float(r.v[i >> 2][i & 3]);
        else if constexpr (__is_same(E, ElemBF16))
            f[i] = __uint_as_float(i & 1 ? r.v[0][i >> 1] & 0xFFFF0000u : r.v[0][i >> 1] << 16);
        else
            f[i] = __half2float(__ushort_as_half((unsigned short)(r.v[0][i >> 1] >> (16 * (i & 1)))));
    }
}

// eight elements that are already rounded to E, stored at row[k0 .. min(k0 + 8, K))
template <typename E>
__device__ __forceinline__ void store8(char *row, int k0, int K, const float (&f)[8]) {
    if (k0 + 8 <= K) {
        u32x4_anywhere *p = reinterpret_cast<u32x4_anywhere *>(row + (int64_t)k0 * Elem<E>::bytes);
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (__is_same(E, ElemF16)) w[i] = (uint32_t)__half_as_ushort(__float2half(f[i]));
            else w[i] = __float_as_uint(f[i]) >> (__is_same(E, ElemBF16) ? 16 : 0);
        }
        if constexpr (Elem<E>::bytes == 4) {
            p[0] = u32x4{w[0], w[1], w[2], w[3]};
            p[1] = u32x4{w[4], w[5], w[6], w[7]};
        } else {
            p[0] = u32x4{w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k0 + i < K) Elem<E>::store1(row, k0 + i, f[i]);
}

// The 16 lanes that share a block (of numbers y * common) find its largest magnitude, then each writes its eight e4m3 bytes and
// the first the scale.
__device__ __forceinline__ void write_block(const float (&y)[8], float common, int sub, uint8_t *q8, float *scale) {
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, ha_abs_bits(y[i]));
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 16));
    const HaFp8Scale s = ha_fp8_scale(top, common);
    *reinterpret_cast<uint2 *>(q8) = make_uint2(ha_fp8x4(y[0] * s.inv, y[1] * s.inv, y[2] * s.inv, y[3] * s.inv),
                                                ha_fp8x4(y[4] * s.inv, y[5] * s.inv, y[6] * s.inv, y[7] * s.inv));
    if (sub == 0) *scale = s.scale;
}

// One block of 128 per 16 lanes, eight elements per lane; blocks of all rows in one flat order, so that narrow rows fill a
// workgroup too.  PAIR: x holds [gate | up] rows of 2 K elements and the block is that of silu(gate) * up.  Bound by memory: SwiGLU of
// 4096 x 14336 58 us (60.6 at a large copy's rate), rows of 8192 x 4096 21 us; 4 x 4096 2.1 us, a launch's length.
template <typename E, bool PAIR>
__global__ __launch_bounds__(256) void rows_fp8_kernel(const char *__restrict__ x, int64_t x_sb, int n_blocks, int kb_count, int K,
                                                       uint8_t *__restrict__ q, int64_t q_sm, float *__restrict__ scales, int64_t s_sm) {
    const int sub = threadIdx.x & 15;
    const int blk = (int)(blockIdx.x * 16u + (threadIdx.x >> 4));
    if (blk >= n_blocks) return;  // whole groups of 16 lanes leave together
    const int m = blk / kb_count, kb = blk - m * kb_count, k0 = kb * HA_FP8_BLOCK + sub * 8;
    const char *row = x + m * x_sb;
    float y[8];
    to_float<E>(load8<E>(row, k0, K), y);
    if constexpr (PAIR) {
        float u[8];
        to_float<E>(load8<E>(row + (int64_t)K * Elem<E>::bytes, k0, K), u);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = ha_silu(y[i]) * u[i];
    }
    write_block(y, 1.0f, sub, q + m * q_sm + k0, scales + m * s_sm + kb);
}

// One workgroup of T threads per row, the row in registers between the sum of squares and the scaling (PER x 8 elements per
// thread).  h = x + residual is rounded to the element type first: what is stored for the next addition is what is normalised.
// h may be stored over x or the residual: every thread has read its elements of both before it stores them.  Bound by memory: 8192 x
// 4096 with a residual 46 us (48.4 at a large copy's rate); 4 x 4096 3.9 us, one row's chain of load, sum, barrier and write.
template <typename E, int T, int PER>
__global__ __launch_bounds__(T) void rmsnorm_fp8_kernel(const char *x, int64_t x_sb, const char *res, int64_t res_sb,
                                                        const char *__restrict__ w, int K, float eps, char *sum_out, int64_t sum_sb,
                                                        uint8_t *__restrict__ q, int64_t q_sm, float *__restrict__ scales, int64_t s_sm) {
    __shared__ float s_sum[T / 64];
    const int tid = threadIdx.x;
    const int64_t m = blockIdx.x;
    float h[PER][8], a = 0.f;
    // the weights are requested with the row, ahead of the sum that the scaling waits for, where registers allow it
    constexpr bool kAhead = PER <= 4;
    Eight<E> ahead[kAhead ? PER : 1];
    if constexpr (kAhead) {
#pragma unroll
        for (int i = 0; i < PER; ++i) ahead[i] = load8<E>(w, (tid + i * T) * 8, K);
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) to_float<E>(load8<E>(x + m * x_sb, (tid + i * T) * 8, K), h[i]);
    if (res) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            float r[8];
            to_float<E>(load8<E>(res + m * res_sb, (tid + i * T) * 8, K), r);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = ha_round_to(h[i][j] + r[j], dtype_of<E>);
        }
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        if (sum_out) store8<E>(sum_out + m * sum_sb, (tid + i * T) * 8, K, h[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) a = fmaf(h[i][j], h[i][j], a);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) a += __shfl_xor(a, o);
    if constexpr (T > 64) {
        if ((tid & 63) == 0) s_sum[tid >> 6] = a;
        __syncthreads();
        a = 0.f;
#pragma unroll
        for (int i = 0; i < T / 64; ++i) a += s_sum[i];
    }
    const float rstd = 1.0f / sqrtf(a / (float)K + eps);
    // Its power of two scales the row exactly; what is left, 1 to 2, is common to every block and only the block's scale takes it.
    // So the numbers carry the product's rounding alone, none in 16 bits, and neither the root's nor its reciprocal's, and as few
    // of them as can be land on the other side of an e4m3 step.  A NaN's power is infinity: the row is NaN.
    const float power = __uint_as_float(__float_as_uint(rstd) & 0x7F800000u);
    const float common = __uint_as_float((__float_as_uint(rstd) & 0x007FFFFFu) | 0x3F800000u);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int k0 = (tid + i * T) * 8;
        if (k0 / HA_FP8_BLOCK * HA_FP8_BLOCK >= K) continue;  // whole groups of 16 lanes: the block lies beyond the row
        float g[8];
        if constexpr (kAhead) to_float<E>(ahead[i], g);
        else to_float<E>(load8<E>(w, k0, K), g);
#pragma unroll
        for (int j = 0; j < 8; ++j) g[j] = h[i][j] * power * g[j];
        if (k0 + 8 > K) {  // 0 * infinity at the padding would be NaN
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k0 + j >= K) g[j] = 0.f;
        }
        write_block(g, common, tid & 15, q + m * q_sm + k0, scales + m * s_sm + k0 / HA_FP8_BLOCK);
    }
}

int check_rows(const void *q, int64_t q_stride_m, const float *scales, int64_t s_stride_m, int M, int K) {
    HA_REQUIRE(M == 0 || (q && scales), HA_ERR_NULL_POINTER, "q/scales is NULL");
    HA_REQUIRE(M >= 0 && K >= 1 && K <= HA_FP8_MAX_K, HA_ERR_BAD_SHAPE, "need M >= 0 rows of K >= 1 elements, K <= %d", HA_FP8_MAX_K);
    const int64_t kb = ha_fp8_blocks(K);
    HA_REQUIRE(q_stride_m >= kb * HA_FP8_BLOCK && s_stride_m >= kb, HA_ERR_BAD_SHAPE,
               "a row of q spans ha_fp8_row_bytes(K) bytes and a row of scales one number per block of 128");
    HA_REQUIRE(ha_fits_launch((M * kb + 15) / 16, 256), HA_ERR_BAD_SHAPE, "too many blocks for one launch");
    HA_REQUIRE(ha_aligned(q, 16) && q_stride_m % 16 == 0 && ha_aligned(scales, 4), HA_ERR_MISALIGNED, "rows of q must be 16-byte aligned");
    return HA_OK;
}

template <bool PAIR>
int launch_rows(const void *x, int64_t x_stride_m, int dtype, int M, int K, void *q, int64_t q_stride_m, float *scales, int64_t s_stride_m,
                void *stream) {
    const int kb = ha_fp8_blocks(K), n = M * kb;
    const unsigned grid = (unsigned)((n + 15LL) / 16);
    const int64_t x_sb = x_stride_m * ha_dtype_bytes(dtype);
#define HA_ROWS(E_)                                                                                                                 \
    hipLaunchKernelGGL((rows_fp8_kernel<E_, PAIR>), dim3(grid), dim3(256), 0, (hipStream_t)stream, (const char *)x, x_sb, n, kb, K, \
                       (uint8_t *)q, q_stride_m, scales, s_stride_m)
    if (dtype == HA_F32) {
        HA_ROWS(ElemF32);
    } else if (dtype == HA_BF16) {
        HA_ROWS(ElemBF16);
    } else {
        HA_ROWS(ElemF16);
    }
#undef HA_ROWS
    HA_CHECK_LAUNCH("rows_fp8_kernel");
    return HA_OK;
}

}  // namespace

extern "C" {

int64_t ha_fp8_row_bytes(int K) { return K >= 1 ? (int64_t)ha_fp8_blocks(K) * HA_FP8_BLOCK : 0; }

int ha_quantize_rows_fp8(const void *x, int64_t x_stride_m, int dtype, int M, int K, void *q, int64_t q_stride_m, float *scales,
                         int64_t scales_stride_m, void *stream) {
    HA_REQUIRE(M == 0 || x, HA_ERR_NULL_POINTER, "x is NULL");
    HA_REQUIRE(dtype == HA_F32 || dtype == HA_BF16 || dtype == HA_F16, HA_ERR_BAD_DTYPE, "unknown dtype %d", dtype);
    int st = check_rows(q, q_stride_m, scales, scales_stride_m, M, K);
    if (st) return st;
    HA_REQUIRE(x_stride_m >= K, HA_ERR_BAD_SHAPE, "x_stride_m smaller than a row");
    HA_REQUIRE(ha_aligned(x, ha_dtype_bytes(dtype)), HA_ERR_MISALIGNED, "x is not aligned to its elements");
    st = ha_require_device();
    if (st || M == 0) return st;
    return launch_rows<false>(x, x_stride_m, dtype, M, K, q, q_stride_m, scales, scales_stride_m, stream);
}

int ha_swiglu_fp8(const void *gate_up, int64_t gate_up_stride_m, int dtype, int M, int F, void *q, int64_t q_stride_m, float *scales,
                  int64_t scales_stride_m, void *stream) {
    HA_REQUIRE(M == 0 || gate_up, HA_ERR_NULL_POINTER, "gate_up is NULL");
    HA_REQUIRE(dtype == HA_F32 || dtype == HA_BF16 || dtype == HA_F16, HA_ERR_BAD_DTYPE, "unknown dtype %d", dtype);
    int st = check_rows(q, q_stride_m, scales, scales_stride_m, M, F);
    if (st) return st;
    HA_REQUIRE(gate_up_stride_m >= 2 * (int64_t)F, HA_ERR_BAD_SHAPE, "a row of gate_up holds 2 F elements");
    HA_REQUIRE(ha_aligned(gate_up, ha_dtype_bytes(dtype)), HA_ERR_MISALIGNED, "gate_up is not aligned to its elements");
    st = ha_require_device();
    if (st || M == 0) return st;
    return launch_rows<true>(gate_up, gate_up_stride_m, dtype, M, F, q, q_stride_m, scales, scales_stride_m, stream);
}

int ha_rmsnorm_fp8(const void *x, int64_t x_stride_m, const void *residual, int64_t residual_stride_m, const void *weight, int dtype, int M,
                   int K, float eps, void *sum_out, int64_t sum_stride_m, void *q, int64_t q_stride_m, float *scales,
                   int64_t scales_stride_m, void *stream) {
    HA_REQUIRE(weight && (M == 0 || x), HA_ERR_NULL_POINTER, "x/weight is NULL");
    HA_REQUIRE(dtype == HA_F32 || dtype == HA_BF16 || dtype == HA_F16, HA_ERR_BAD_DTYPE, "unknown dtype %d", dtype);
    int st = check_rows(q, q_stride_m, scales, scales_stride_m, M, K);
    if (st) return st;
    HA_REQUIRE(K <= 65536, HA_ERR_BAD_SHAPE, "rows of up to 65536 elements");
    HA_REQUIRE(ha_fits_launch(M, K <= 512 ? 64 : K <= 8192 ? 256 : 1024), HA_ERR_BAD_SHAPE, "too many rows for one launch");
    HA_REQUIRE(x_stride_m >= K && (!residual || residual_stride_m >= K) && (!sum_out || sum_stride_m >= K) && eps >= 0.f, HA_ERR_BAD_SHAPE,
               "strides smaller than a row, or a negative eps");
    const int es = ha_dtype_bytes(dtype);
    HA_REQUIRE(ha_aligned(x, es) && ha_aligned(residual, es) && ha_aligned(weight, es) && ha_aligned(sum_out, es), HA_ERR_MISALIGNED,
               "pointers are not aligned to their elements");
    st = ha_require_device();
    if (st || M == 0) return st;
#define HA_NORM(E_, T_, P_)                                                                                                          \
    hipLaunchKernelGGL((rmsnorm_fp8_kernel<E_, T_, P_>), dim3((unsigned)M), dim3(T_), 0, (hipStream_t)stream, (const char *)x,       \
                       x_stride_m * es, (const char *)residual, residual_stride_m * es, (const char *)weight, K, eps, (char *)sum_out,    \
                       sum_stride_m * es, (uint8_t *)q, q_stride_m, scales, scales_stride_m)
#define HA_NORM_SIZE(E_)                            \
    do {                                                \
        if (K <= 512) HA_NORM(E_, 64, 1);           \
        else if (K <= 2048) HA_NORM(E_, 256, 1);    \
        else if (K <= 4096) HA_NORM(E_, 256, 2);    \
        else if (K <= 8192) HA_NORM(E_, 256, 4);    \
        else if (K <= 16384) HA_NORM(E_, 1024, 2);  \
        else HA_NORM(E_, 1024, 8);                  \
    } while (0)
    if (dtype == HA_F32) {
        HA_NORM_SIZE(ElemF32);
    } else if (dtype == HA_BF16) {
        HA_NORM_SIZE(ElemBF16);
    } else {
        HA_NORM_SIZE(ElemF16);
    }
#undef HA_NORM_SIZE
#undef HA_NORM
    HA_CHECK_LAUNCH("rmsnorm_fp8_kernel");
    return HA_OK;
}

}  // extern "C"
