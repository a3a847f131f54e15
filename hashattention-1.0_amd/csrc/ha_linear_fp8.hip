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
// keeps its sums in fp32 (1.2e-8 on the same numbers), at half the 8-bit rate plus one conversion per two numbers.  So: fp32
// results and up to 16 rows, where the stream of weights is the bound and the conversions cost nothing, run on the bf16
// instruction; 16-bit results of more rows on the 8-bit one: a bf16 result's own rounding (2^-9 of the value) is 130 times the loss on
// normal numbers and 20 times that on widely spread ones, an fp16 result's (2^-12) 16 and 2.4 times.  Both are figures of a result that is
// not small against its products; where they cancel, the loss is up to 2^-10 of the sum of their magnitudes, and fp32 out avoids it.
//
//   ha_weight_fp8_bytes / ha_weight_fp8_scales / ha_pack_weight_fp8   the packed weights
//   ha_linear_fp8                                                     the product, residual or SwiGLU behind
#include "ha_fp8.h"

namespace {

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
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
__device__ __forceinline__ Wide widen(const u32x4 &a, const u32x4 &b) {
    return {{widen8(a.x, a.y), widen8(a.z, a.w), widen8(b.x, b.y), widen8(b.z, b.w)}};
}
__device__ __forceinline__ f32x4 block_sum(const Wide &w, const Wide &x) {
    f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], c, 0, 0, 0);
    return c;
}

// An operand of a block of 128 inputs, made of a lane's two pieces.  EXACT: bf16 matrix instructions on widened numbers; otherwise the
// 8-bit one (see the top of this file).
template <bool EXACT>
struct Operand;
template <>
struct Operand<false> {
    i32x8 v;
    __device__ __forceinline__ void take(const u32x4 &a, const u32x4 &b) {
        v = __builtin_bit_cast(i32x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // constant zero scale operands select the instruction without block exponents
    __device__ static __forceinline__ f32x4 product(const Operand &w, const Operand &x) {
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
    }
};
template <>
struct Operand<true> {
    Wide v;
    __device__ __forceinline__ void take(const u32x4 &a, const u32x4 &b) { v = widen(a, b); }
    __device__ static __forceinline__ f32x4 product(const Operand &w, const Operand &x) { return block_sum(w.v, x.v); }
};

struct Epilogue {
    const void *res;
    int64_t res_sm;
    void *out;
    int64_t out_sm;
    int out_dtype;
    bool wide, wide8;  // four neighbouring columns of out and residual, eight of out are one aligned access
};

// y += residual[m, n .. min(n + 4, cols))
__device__ __forceinline__ void add_residual(const Epilogue &ep, int64_t m, int n, int cols, f32x4 &y) {
    if (ep.wide && n + 4 <= cols) {
        if (ep.out_dtype == HA_F32) {
            y += *reinterpret_cast<const f32x4 *>((const float *)ep.res + m * ep.res_sm + n);
        } else {
            const uint2 b = *reinterpret_cast<const uint2 *>((const uint16_t *)ep.res + m * ep.res_sm + n);
            const uint32_t w[4] = {b.x & 0xFFFFu, b.x >> 16, b.y & 0xFFFFu, b.y >> 16};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                y[i] += ep.out_dtype == HA_BF16 ? __uint_as_float(w[i] << 16) : __half2float(__ushort_as_half((unsigned short)w[i]));
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < cols) y[i] += ha_load_elem(ep.res, m * ep.res_sm + n + i, ep.out_dtype);
}

// four results as 16-bit numbers
__device__ __forceinline__ uint2 narrow4(const f32x4 &y, int dtype) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = dtype == HA_BF16 ? ha_f32_to_bf16_bits(y[i]) : (uint32_t)__half_as_ushort(__float2half(y[i]));
    return make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}

// fp32 out[m, n .. min(n + 4, cols)) = y (+ residual)
__device__ __forceinline__ void store4(const Epilogue &ep, int64_t m, int n, int cols, f32x4 y) {
    if (ep.res) add_residual(ep, m, n, cols, y);
    float *o = (float *)ep.out + m * ep.out_sm + n;
    if (ep.wide && n + 4 <= cols) {
        *reinterpret_cast<f32x4 *>(o) = y;
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n + i < cols) o[i] = y[i];
}

// The waves' sums of NT tiles from nt on (s_c[wave][weight row][row of x]) joined, finished and stored by the whole workgroup.
template <int NWAVE, int NT, int MT, bool GLU>
__device__ __forceinline__ void join_waves(const float (&s_c)[NWAVE][16 * NT][16 * MT + 1], const Epilogue &ep, int nt, int m0, int M, int N) {
    const int tid = threadIdx.x;
    auto total = [&](int row, int mm) {
        float y = 0.f;
#pragma unroll
        for (int w = 0; w < NWAVE; ++w) y += s_c[w][row][mm];
        return y;
    };
    if constexpr (GLU) {
        for (int t = tid; t < 8 * NT * 16 * MT; t += NWAVE * 64) {
            const int mm = t / (8 * NT), c = t % (8 * NT), col = 8 * nt + c;
            if (m0 + mm >= M || col >= N / 2) continue;
            const int row = (c >> 3) * 16 + (c & 7);
            const float gate = total(row, mm);
            ha_store_elem(ep.out, (m0 + mm) * ep.out_sm + col, ha_silu(gate) * total(row + 8, mm), ep.out_dtype);
        }
    } else {
        for (int t = tid; t < 16 * NT * 16 * MT; t += NWAVE * 64) {
            const int mm = t / (16 * NT), c = t % (16 * NT), n = 16 * nt + c;
            if (m0 + mm >= M || n >= N) continue;
            float y = total(c, mm);
            if (ep.res) y += ha_load_elem(ep.res, (m0 + mm) * ep.res_sm + n, ep.out_dtype);
            ha_store_elem(ep.out, (m0 + mm) * ep.out_sm + n, y, ep.out_dtype);
        }
    }
}

// ---- any size: NT tiles of 16 weight rows and 16 MT rows of x per workgroup, straight from memory to registers
//
// The waves cut K into slices and walk them in groups of PF blocks, weights and rows of x requested together, a group ahead, without
// a barrier; their sums are joined through LDS.  For rows too long for registers: up to 16 rows, 17 to 32 where the tiles need no cut
// of K, and rows of x so far apart that a group's positions pass 32 bits.  NT and MT set how often x and the weights are read.
// Bound by the stream of weights: 4 rows, 4096 x 14336, 11.8 us (5.0 TB/s; 9.7 at the rate of a plain read); 16 rows 15.9 us, the
// rows of x beside it.
template <int NWAVE, int PF, int NT, int MT, bool EXACT, bool GLU>
__global__ __launch_bounds__(NWAVE * 64) void linear_fp8_stream_kernel(const uint8_t *__restrict__ x, int64_t x_sm, const float *__restrict__ xs,
                                                                       int64_t xs_sm, const uint8_t *__restrict__ tiles,
                                                                       const float *__restrict__ ws, Epilogue ep, int M, int N, int kb_count,
                                                                       int n_tiles, int groups_m) {
    __shared__ float s_c[NWAVE][16 * NT][16 * MT + 1];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, r = lane & 15, g = lane >> 4;
    // workgroups go to the XCDs in turn: the groups of rows that take the same tiles share an XCD and its L2
    const int turn = (int)(blockIdx.x >> 3), m0 = turn % groups_m * 16 * MT, nt = (turn / groups_m * 8 + (int)(blockIdx.x & 7)) * NT;
    if (nt >= n_tiles) return;
    const int per = ((kb_count + NWAVE - 1) / NWAVE + PF - 1) / PF * PF, begin = wave * per, end = min(begin + per, kb_count);
    // rows beyond M and tiles beyond the matrix are read as the last ones; what they give is not stored
    const u32x4 *tp[NT];
    const float *wsp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t tile = (int64_t)min(nt + j, n_tiles - 1) * kb_count;
        tp[j] = reinterpret_cast<const u32x4 *>(tiles + tile * kTileBytes);
        wsp[j] = ws + tile * 2;
    }
    const uint8_t *xp[MT];
    const float *xsp[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int64_t m = min(m0 + 16 * t + r, M - 1);
        xp[t] = x + m * x_sm + g * 16;
        xsp[t] = xs + m * xs_sm;
    }
    struct Group {
        u32x4 wa[PF][NT], wb[PF][NT], xa[PF][MT], xb[PF][MT];
        float ws[PF][NT], xs[PF][MT];
    };
    // blocks beyond the slice are read as its last one and count nothing
    auto fetch = [&](Group &f, int kb0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int kb = min(kb0 + i, end - 1);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                f.wa[i][j] = __builtin_nontemporal_load(tp[j] + (int64_t)kb * (kTileBytes / 16) + lane);
                f.wb[i][j] = __builtin_nontemporal_load(tp[j] + (int64_t)kb * (kTileBytes / 16) + 64 + lane);
                f.ws[i][j] = wsp[j][2 * kb + (g >> 1)];
            }
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                f.xa[i][t] = *reinterpret_cast<const u32x4 *>(xp[t] + kb * HA_FP8_BLOCK);
                f.xb[i][t] = *reinterpret_cast<const u32x4 *>(xp[t] + kb * HA_FP8_BLOCK + 64);
                f.xs[i][t] = xsp[t][kb];
            }
        }
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[j][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const Group &f, int count) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            if (i < count) {
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    Operand<EXACT> w, v;
                    w.take(f.wa[i][j], f.wb[i][j]);
#pragma unroll
                    for (int t = 0; t < MT; ++t) {
                        v.take(f.xa[i][t], f.xb[i][t]);
                        const f32x4 part = Operand<EXACT>::product(w, v);
                        const float s = f.xs[i][t] * f.ws[i][j];
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[j][t][e] = fmaf(part[e], s, acc[j][t][e]);
                    }
                }
            }
        }
    };
    if (begin < end) {
        Group now, next;
        fetch(now, begin);
        int kb = begin;
        // the loop always requests: behind a request that may not have been made, the compiler waits for all of them
        for (; kb + PF < end; kb += PF) {
            fetch(next, kb + PF);
            __builtin_amdgcn_sched_barrier(0);  // in front of the products: the compiler would move the requests behind them
            multiply(now, PF);
            now = next;
        }
        multiply(now, end - kb);
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_c[wave][16 * j + 4 * g + i][16 * t + r] = acc[j][t][i];
    __syncthreads();
    join_waves<NWAVE, NT, MT, GLU>(s_c, ep, nt, m0, M, N);
}

// ---- few rows: x in registers, the weights streamed once
//
// The waves of a workgroup cut K into slices of KW blocks; each keeps its slice of 16 MT rows of x in registers (as e4m3, 8
// registers per block and 16 rows; widened when used) and walks the weight tiles blockIdx, blockIdx + step, ...: per tile KW
// blocks of 2 KiB, consecutive in memory, requested PF blocks ahead.  The waves' sums are joined through LDS.  What bounds it is
// the stream of weights (16 rows, 28672 x 4096 with SwiGLU, 20.4 us, 5.8 TB/s); the conversions (16 per block and 16 rows) and the
// matrix instructions run under it.  With more rows it is the start, x out of L2 into every workgroup, and about 2.6 us per tile
// behind it (6144 x 4096, three tiles: 128 rows 13.2 us).
template <int NWAVE, int KW, int PF, int MT, bool WIDE, bool EXACT, bool GLU>
__global__ __launch_bounds__(NWAVE * 64) void linear_fp8_rows_kernel(const uint8_t *__restrict__ x, int64_t x_sm, const float *__restrict__ xs,
                                                                     int64_t xs_sm, const uint8_t *__restrict__ tiles,
                                                                     const float *__restrict__ ws, Epilogue ep, int M, int N, int kb_count,
                                                                     int n_tiles, int groups_m) {
    static_assert(KW % PF == 0, "a slice is whole groups of blocks");
    __shared__ float s_c[2][NWAVE][16][16 * MT + 1];
    __shared__ u32x4 s_x[NWAVE][128];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, r = lane & 15, g = lane >> 4;
    // workgroups go to the XCDs in turn: the groups of rows that walk the same tiles share an XCD and its L2
    const int turn = (int)(blockIdx.x >> 3), step = (int)(gridDim.x / (unsigned)groups_m);
    const int m0 = turn % groups_m * 16 * MT, kb0 = wave * KW;
    int nt = turn / groups_m * 8 + (int)(blockIdx.x & 7);

    // Tiles are requested without a condition (behind a request that may not have been made, the compiler waits for all of them):
    // blocks beyond K are read as the last one and count nothing, rows beyond M as the last one and are not stored.
    struct Group {
        u32x4 a[PF], b[PF];
        float s[PF];
    };
    auto fetch = [&](Group &w, int nt, int j0) __attribute__((always_inline)) {
        const int64_t tile = (int64_t)nt * kb_count;
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            const int kb = kb0 + j0 + i, from = min(kb, kb_count - 1);
            const u32x4 *tp = reinterpret_cast<const u32x4 *>(tiles + (tile + from) * kTileBytes) + lane;
            w.a[i] = __builtin_nontemporal_load(tp);
            w.b[i] = __builtin_nontemporal_load(tp + 64);
            w.s[i] = ws[(tile + from) * 2 + (g >> 1)];
        }
    };
    if (nt >= n_tiles) return;
    Group now, next;
    fetch(now, nt, 0);  // the first weights are on their way before x is set up
    // Rows of x are read as whole lines of 128 bytes, eight to a load, and turned through LDS into the operand's order (row r: chunks g
    // and 4 + g), two KiB per wave; chunk c of row r lies in place c ^ (r & 7) of its line, which keeps both sides free of bank
    // conflicts.  Read in the operand's order, 16 rows at a time, a load takes half lines of twice as many, and x is what a
    // workgroup waits for first.  A row's scales are consecutive: one load for the slice, moved where the slice ends behind K.
    // (6144 x 4096, 128 rows: 19.3 us with x in the operand's order and scales one by one, 16.0 with the scales' load, 13.2 with both.)
    u32x4 xa[KW][MT], xb[KW][MT];
    float xsc[KW][MT];
#pragma unroll
    for (int j = 0; j < KW; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const uint8_t *xp = x + min(kb0 + j, kb_count - 1) * HA_FP8_BLOCK + (lane & 7) * 16;
            xa[j][t] = *reinterpret_cast<const u32x4 *>(xp + (int64_t)min(m0 + 16 * t + (lane >> 3), M - 1) * x_sm);
            xb[j][t] = *reinterpret_cast<const u32x4 *>(xp + (int64_t)min(m0 + 16 * t + 8 + (lane >> 3), M - 1) * x_sm);
        }
    const int s_from = max(min(kb0, kb_count - KW), 0), s_past = kb0 - s_from;
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const float *sp = xs + (int64_t)min(m0 + 16 * t + r, M - 1) * xs_sm + s_from;
        float v[KW];
        if constexpr (KW == 1) {
            v[0] = sp[0];
        } else {
            typedef float run __attribute__((ext_vector_type(KW), aligned(4)));
            const run f = *reinterpret_cast<const run *>(sp);
#pragma unroll
            for (int j = 0; j < KW; ++j) v[j] = f[j];
        }
#pragma unroll
        for (int j = 0; j < KW; ++j) {
            xsc[j][t] = v[j];
#pragma unroll
            for (int d = 1; j + d < KW; ++d)
                if (s_past == d) xsc[j][t] = v[j + d];
        }
    }
    u32x4 *turn_x = s_x[wave];
#pragma unroll
    for (int j = 0; j < KW; ++j)
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            turn_x[(lane >> 3) * 8 + ((lane & 7) ^ (lane >> 3))] = xa[j][t];
            turn_x[(8 + (lane >> 3)) * 8 + ((lane & 7) ^ (lane >> 3))] = xb[j][t];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the wave's LDS accesses stay in this order
            __builtin_amdgcn_wave_barrier();
            xa[j][t] = turn_x[r * 8 + (g ^ (r & 7))];
            xb[j][t] = turn_x[r * 8 + ((4 + g) ^ (r & 7))];
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    f32x4 acc[MT];
    int side = 0;
    auto multiply = [&](const Group &w, int j0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < PF; ++i) {
            Operand<EXACT> wo, v;
            wo.take(w.a[i], w.b[i]);
            const bool counts = kb0 + j0 + i < kb_count;
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                v.take(xa[j0 + i][t], xb[j0 + i][t]);
                const f32x4 part = Operand<EXACT>::product(wo, v);
                const float s = counts ? xsc[j0 + i][t] * w.s[i] : 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(part[e], s, acc[t][e]);
            }
        }
    };
    // one tile: its first group is in `now`; the first group of `then` (if any) is there afterwards
    auto tile = [&](int nt, int then, bool more) __attribute__((always_inline)) {
        if constexpr (EXACT && !WIDE) {  // the compiler would widen x once, in front of the loop, at twice the registers
#pragma unroll
            for (int j = 0; j < KW; ++j)
#pragma unroll
                for (int t = 0; t < MT; ++t)
                    asm volatile("" : "+v"(xa[j][t]), "+v"(xb[j][t]));
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j0 = 0; j0 < KW; j0 += PF) {
            if (j0 + PF < KW) fetch(next, nt, j0 + PF);
            else if (more) fetch(next, then, 0);
            __builtin_amdgcn_sched_barrier(0);  // in front of the products: the compiler would move the requests behind them
            multiply(now, j0);
            now = next;
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) s_c[side][wave][4 * g + i][16 * t + r] = acc[t][i];
        __syncthreads();
        join_waves<NWAVE, 1, MT, GLU>(s_c[side], ep, nt, m0, M, N);
        side ^= 1;  // the next tile's sums go to the other buffer; a wave is back at this one only behind the barrier in between
    };
    for (; nt + step < n_tiles; nt += step) tile(nt, nt + step, true);
    tile(nt, nt, false);
}

// ---- many rows: tiles of BN weight rows x BM rows of x per workgroup, staged through LDS
//
// WN x WM waves of TN x TM operand tiles each (16 weight rows, 16 rows of x).  Everything a block of 128 inputs needs travels
// from memory straight to LDS (one KiB per request and wave).  4096 x 28672 x 4096 in 480 - 500 us, 2.0 PFLOP/s, where no unit is busy
// all the time: matrix cores 50 % of the cycles, other vector instructions (the blocks' scales, a multiply-add per result and block)
// 36 %, LDS reads 23 %; every wave spends 29 % of its life at the two barriers of a block.  Weights lie there in the order the matrix instruction takes
// them, lane l's 16 bytes at l * 16.  Rows of x arrive as whole 128-byte lines, eight to a request; the 16-byte chunk c of row r
// sits in place c ^ (r & 7) of its line - each lane asks for the chunk that belongs in its place - so that the eight lanes that an
// LDS read serves at a time, same chunk of eight rows, meet eight different bank groups.
//
// Two buffers, each in two parts: x with the first half of every wave's weight tiles, and the second half.  A part is requested
// as soon as all waves have read the part of two blocks before out of its place, half a block's time after the other: between
// its request and its use lie one and a half blocks' time, and three quarters of the buffers are always on their way.
// Requests from memory straight to LDS: lane l's 16 (4) bytes from base + offset + from, and i * kStep more for the i-th of a call,
// land at lds + l * 16 (l * 4) + i * kStep; `from` and lds are uniform over the wave.  A buffer resource takes its base from four
// scalar registers and `from` from a fifth, so that a request costs no address arithmetic; the instruction's own offset counts
// for both sides, which is why targets of one call lie kStep apart.
// Inline assembly, because the compiler would wait for all of them in front of every LDS read it cannot tell from their target;
// the waits are written by hand (requests_arrived).  M0 holds the LDS address; nothing else in the kernel uses M0.
__device__ __forceinline__ u32x4 resource(const void *base) {  // uniform base; every access of this file is in bounds by itself
    const uint64_t b = (uint64_t)base;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b), (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32)),
                 0xFFFFFFFFu, 0x00020000u};
}
__device__ __forceinline__ void request16x2(u32x4 res, uint32_t offset, uint32_t from, uint32_t lds) {  // kStep 1024
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %3 offen lds\n\t"
                 "buffer_load_dwordx4 %0, %1, %3 offen offset:1024 lds"
                 ::"v"(offset), "s"(res), "s"(lds), "s"(from)
                 : "memory");
}
// the same with an offset of its own for each of the two, of which the first lies `first` behind lds
template <int FIRST>
__device__ __forceinline__ void request16_pair(u32x4 res, uint32_t offset0, uint32_t offset1, uint32_t from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, %4 offen offset:%5 lds\n\t"
                 "buffer_load_dwordx4 %1, %2, %4 offen offset:%6 lds"
                 ::"v"(offset0), "v"(offset1), "s"(res), "s"(lds), "s"(from), "n"(FIRST), "n"(FIRST + 1024)
                 : "memory");
}
__device__ __forceinline__ void request4(u32x4 res, uint32_t offset, uint32_t from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, %3 offen lds" ::"v"(offset), "s"(res), "s"(lds), "s"(from) : "memory");
}
// Waits until at most YOUNGER of the wave's requests are outstanding (they arrive in the order they were made) and every wave
// has come here; all LDS reads of the wave have arrived too.  The count relies on the loop having no other vector memory access:
// no global load and no spilled register.  -DHASHATTN_STAGE_WAIT_ALL builds the conservative form, which must give the same bits.
template <int YOUNGER>
__device__ __forceinline__ void requests_arrived() {
#ifdef HASHATTN_STAGE_WAIT_ALL
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#else
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(YOUNGER) : "memory");
#endif
    __syncthreads();
}

template <int WN, int WM, int TN, int TM, int AHEAD, bool EXACT, bool GLU, bool SPLIT>
__global__ __launch_bounds__(WN *WM * 64) void linear_fp8_tiled_kernel(const uint8_t *__restrict__ x, int64_t x_sm,
                                                                       const float *__restrict__ xs, int64_t xs_sm,
                                                                       const uint8_t *__restrict__ tiles, const float *__restrict__ ws,
                                                                       Epilogue ep, int M, int N, int kb_count, int n_tiles, int tiles_n,
                                                                       int tiles_m, int per_xcd, int per_split, float *__restrict__ partial) {
    constexpr int NW = WN * WM, BN = 16 * TN * WN, BM = 16 * TM * WM, TH = TN / 2;
    constexpr int kWBytes = BN * HA_FP8_BLOCK, kXBytes = BM * HA_FP8_BLOCK, kBuffer = kWBytes + kXBytes;
    constexpr int kHalfPieces = kWBytes / 2048 / NW, kXPieces = kXBytes / 1024 / NW;  // requests per wave: half of the weights, x
    constexpr int kFirst = kXPieces + kHalfPieces + 2, kSecond = kHalfPieces;          // requests per wave and part (two for the scales)
    static_assert(kWBytes % (2048 * NW) == 0 && kXBytes % (1024 * NW) == 0 && BM <= 64 * NW && BM % 64 == 0, "pieces deal out evenly");
    static_assert(TN % 2 == 0 && 16 * TN <= HA_FP8_BLOCK, "one weight scale per wave, half and block");
    __shared__ __attribute__((aligned(1024))) uint8_t s_buf[2][kBuffer];
    __shared__ float s_xs[2][BM], s_ws[2][NW * 64];
    // Workgroups go to the XCDs in turn: XCD j takes a run of tiles, four tiles of x wide and then along N, so that the 32 CUs
    // that share an L2 work on a compact block of the result.
    int linear = (int)(blockIdx.x & 7) * per_xcd + (int)(blockIdx.x >> 3), kb_begin = 0, kb_end = kb_count;
    int64_t split = 0;
    if constexpr (SPLIT) {  // the splits of a tile share an XCD, one behind the other
        const int all = tiles_n * tiles_m;
        split = linear / all;
        linear -= (int)split * all;
        kb_begin = (int)split * per_split;
        kb_end = min(kb_begin + per_split, kb_count);
        if (kb_begin >= kb_end) return;
    } else {
        if (linear >= tiles_n * tiles_m) return;
    }
    const int band = linear / (4 * tiles_n), in_band = linear - band * 4 * tiles_n, rows_in_band = min(4, tiles_m - 4 * band);
    const int bm = 4 * band + in_band % rows_in_band, bn = in_band / rows_in_band;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wave % WN, wm = wave / WN;
    const int m0 = bm * BM, nt0 = bn * (BN / 16);

    // rows and tiles beyond the matrices are read as their last ones; what they give is not stored
    static_assert(kXPieces == 4 && kHalfPieces == 2, "requests are made by two");
    const u32x4 x_res = resource(x + (int64_t)m0 * x_sm - 4096), xs_res = resource(xs + (int64_t)m0 * xs_sm);
    const u32x4 w_res = resource(tiles + (int64_t)nt0 * kb_count * kTileBytes);
    // all tiles of a wave lie in one block of 128 weight rows (glu: one of gate and one of up): one scale per lane and block of K
    const u32x4 ws_res = resource(ws + (int64_t)min(nt0 + wn * TN, n_tiles - 1) * kb_count * 2);
    uint32_t x_off[4], w_off[2], w_at[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 4096 - 1024 i: what the resource's base and the request's own offset take away and add
        const int row = (wave * 4 + i) * 8 + (lane >> 3);
        x_off[i] = (uint32_t)min(row, M - 1 - m0) * (uint32_t)x_sm + ((lane ^ row) & 7) * 16 + 4096 - 1024 * i;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // the wave's tile of each half
        const int tile = wave / TH * TN + h * TH + wave % TH;
        w_at[h] = tile * kTileBytes;
        w_off[h] = (uint32_t)min(tile, n_tiles - 1 - nt0) * (uint32_t)kb_count * kTileBytes + lane * 16;
    }
    const uint32_t xs_off = (uint32_t)min((wave % (BM / 64)) * 64 + lane, M - 1 - m0) * (uint32_t)xs_sm * 4u, ws_off = (g >> 1) * 4u;
    const uint32_t lds_buf = (uint32_t)(uintptr_t)&s_buf[0][0], lds_xs = (uint32_t)(uintptr_t)&s_xs[0][0], lds_ws = (uint32_t)(uintptr_t)&s_ws[0][0];
    // kb: the place; from min(kb, last of the range), so that the loop's requests (hence its waits) are the same in every turn
    auto request_half = [&](int kb, int h) {
        request16x2(w_res, w_off[h], min(kb, kb_end - 1) * kTileBytes, lds_buf + (kb & 1) * kBuffer + w_at[h]);
    };
    auto request_x0 = [&](int kb) {
        request16_pair<0>(x_res, x_off[0], x_off[1], min(kb, kb_end - 1) * HA_FP8_BLOCK, lds_buf + (kb & 1) * kBuffer + kWBytes + wave * 4096);
    };
    auto request_x1 = [&](int kb) {
        request16_pair<2048>(x_res, x_off[2], x_off[3], min(kb, kb_end - 1) * HA_FP8_BLOCK, lds_buf + (kb & 1) * kBuffer + kWBytes + wave * 4096);
    };
    auto request_scales = [&](int kb) {
        request4(xs_res, xs_off, min(kb, kb_end - 1) * 4, lds_xs + ((kb & 1) * BM + wave % (BM / 64) * 64) * 4);
        request4(ws_res, ws_off, min(kb, kb_end - 1) * 8, lds_ws + ((kb & 1) * NW + wave) * 256);
    };

    f32x4 acc[TN][TM];
#pragma unroll
    for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{0.f, 0.f, 0.f, 0.f};
    // LDS addresses of a wave's operands within a buffer
    const uint32_t x_first = kWBytes + (wm * TM * 16 + r) * HA_FP8_BLOCK + ((g ^ r) & 7) * 16, x_second = x_first ^ 64;
    const uint32_t w_first = wn * TN * kTileBytes + lane * 16;
    constexpr int kAhead = AHEAD, kRing = kAhead + 1;  // tiles of weights read ahead of the one in use
    // The tiles at which a block's requests are made: spread out (all of them right behind the barrier, from all waves at once,
    // 4096 x 28672 x 4096 took 579 us against 550).
    constexpr int kX1 = TN == 8 ? 3 : 1, kScales = TN == 8 ? 4 : 2, kHalf0 = TN == 8 ? 5 : 2;
    static_assert(TH - kAhead <= kX1 && kX1 <= kScales && kScales <= kHalf0 && kHalf0 <= TN - kAhead, "the order that the waits count on");
    Operand<EXACT> xo[TM], wo[kRing];
    f32x4 part[2][TM];
    float s[TM], s_next[TM + 1];  // of the next block as they lie in LDS: rows of x, weights
    auto load_row = [&](int kb, int u) {
        const uint8_t *b = &s_buf[0][0] + (kb & 1) * kBuffer + u * kTileBytes;
        xo[u].take(*reinterpret_cast<const u32x4 *>(b + x_first), *reinterpret_cast<const u32x4 *>(b + x_second));
    };
    auto load_scales = [&](int kb) {
        s_next[TM] = s_ws[kb & 1][wave * 64 + lane];
#pragma unroll
        for (int u = 0; u < TM; ++u) s_next[u] = s_xs[kb & 1][(wm * TM + u) * 16 + r];
    };
    auto load_weights = [&](Operand<EXACT> &w, int kb, int t) {
        const uint8_t *b = &s_buf[0][0] + (kb & 1) * kBuffer + w_first + t * kTileBytes;
        w.take(*reinterpret_cast<const u32x4 *>(b), *reinterpret_cast<const u32x4 *>(b + 1024));
    };
    static_assert(TN % kRing == 0 && kAhead < TH, "a block ends on the operand register it began with; its halves are further apart");
    // the order of requests: of every block x, scales, first half, then the second half
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        request_x0(kb_begin + i);
        request_x1(kb_begin + i);
        request_scales(kb_begin + i);
        request_half(kb_begin + i, 0);
        request_half(kb_begin + i, 1);
    }
    requests_arrived<kFirst + 2 * kSecond>();
#pragma unroll
    for (int t = 0; t < kAhead; ++t) load_weights(wo[t], kb_begin, t);
#pragma unroll
    for (int u = 0; u < TM; ++u) load_row(kb_begin, u);
    load_scales(kb_begin);
    // One block of 128 inputs per turn: TN x TM matrix instructions, the multiply-adds of a tile under those of the next one, weights
    // read from LDS kAhead tiles ahead, a row of the next block's x as soon as its last instruction is issued.
    for (int kb = kb_begin; kb < kb_end; ++kb) {
#pragma unroll
        for (int u = 0; u < TM; ++u) s[u] = s_next[u] * s_next[TM];
#pragma unroll
        for (int t = 0; t < TN; ++t) {
            if (t == TH - kAhead) {
                // every wave has x and the first half of this block's weights in registers: the block after next takes their
                // place.  Arrived: the second half of this block.
                requests_arrived<kFirst + kSecond>();
                request_x0(kb + 2);
            }
            if (t == kX1) request_x1(kb + 2);
            if (t == kScales) request_scales(kb + 2);
            if (t == kHalf0) request_half(kb + 2, 0);
            // every wave has the second half in registers too.  Arrived: x and the first half of the next block.
            if (t == TN - kAhead) requests_arrived<kFirst + kSecond>();
            if (t == TN - 1) request_half(kb + 2, 1);
            if (t + kAhead < TN) load_weights(wo[(t + kAhead) % kRing], kb, t + kAhead);
            else load_weights(wo[(t + kAhead) % kRing], kb + 1, t + kAhead - TN);
            if (t == TN - 1) load_scales(kb + 1);
#pragma unroll
            for (int u = 0; u < TM; ++u) {
                part[t & 1][u] = Operand<EXACT>::product(wo[t % kRing], xo[u]);
                if (t == TN - 1) load_row(kb + 1, u);
                if (t > 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[t - 1][u][i] = fmaf(part[(t - 1) & 1][u][i], s[u], acc[t - 1][u][i]);
                }
                __builtin_amdgcn_sched_barrier(0);  // as written: the compiler would hoist the LDS reads of all tiles and spill
            }
        }
#pragma unroll
        for (int u = 0; u < TM; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[TN - 1][u][i] = fmaf(part[(TN - 1) & 1][u][i], s[u], acc[TN - 1][u][i]);
    }
    requests_arrived<0>();

    // acc[t][u][i]: weight row 4 g + i of tile t, row 16 u + r of x
    if constexpr (SPLIT) {  // the split's sums in tile order, [split][m][16 n_tiles]: join_splits finishes them
        const int64_t width = 16LL * n_tiles;
#pragma unroll
        for (int u = 0; u < TM; ++u) {
            const int m = m0 + (wm * TM + u) * 16 + r;
            if (m >= M) continue;
            float *row = partial + (split * M + m) * width + (nt0 + wn * TN) * 16 + 4 * g;
#pragma unroll
            for (int t = 0; t < TN; ++t)
                if (nt0 + wn * TN + t < n_tiles) *reinterpret_cast<f32x4 *>(row + 16 * t) = acc[t][u];
        }
        return;
    }
    constexpr int BO = GLU ? BN / 2 : BN;  // columns of out per workgroup
    const int n_out = GLU ? N / 2 : N, n0 = bn * BO;
    auto each = [&](auto put) {
#pragma unroll
        for (int u = 0; u < TM; ++u)
#pragma unroll
            for (int t = 0; t < TN; ++t) {
                f32x4 y = acc[t][u];
                int col = (wn * TN + t) * 16 + 4 * g;
                if constexpr (GLU) {  // gate in lanes 0 - 31, up in lanes 32 - 63
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float up = __shfl_xor(acc[t][u][i], 32);
                        y[i] = ha_silu(acc[t][u][i]) * up;
                    }
                    col = (wn * TN + t) * 8 + 4 * g;
                    if (g >= 2) continue;
                }
                put((wm * TM + u) * 16 + r, col, y);
            }
    };
    if (ep.out_dtype == HA_F32) {
        each([&](int row, int col, f32x4 y) {
            if (m0 + row < M && n0 + col < n_out) store4(ep, m0 + row, n0 + col, n_out, y);
        });
        return;
    }
    // 16-bit results leave through LDS, so that whole lines are written: a wave's registers hold four columns of sixteen rows.
    // The 16-byte piece c of row m sits in place c ^ (m & 15), within the row's power of two of pieces: the sixteen rows a wave
    // stores at a time meet different banks.
    uint8_t *tile = &s_buf[0][0];
    static_assert(BM * BO * 2 <= 2 * kBuffer, "the result fits where the operands were");
    constexpr int kRowPieces = BO / 8, kTurn = (kRowPieces < 16 ? kRowPieces : 16) - 1;
    static_assert((kRowPieces & (kRowPieces - 1)) == 0, "pieces turn within their row");
    each([&](int row, int col, f32x4 y) {
        if (ep.res) add_residual(ep, m0 + row, n0 + col, (m0 + row < M) ? n_out : 0, y);
        *reinterpret_cast<uint2 *>(tile + row * (BO * 2) + (((col >> 3) ^ (row & kTurn)) * 16) + (col & 4) * 2) = narrow4(y, ep.out_dtype);
    });
    __syncthreads();
    for (int i = tid; i < BM * kRowPieces; i += NW * 64) {
        const int row = i / kRowPieces, c = i % kRowPieces, n = n0 + c * 8;
        if (m0 + row >= M || n >= n_out) continue;
        const uint4 v = *reinterpret_cast<const uint4 *>(tile + row * (BO * 2) + ((c ^ (row & kTurn)) * 16));
        uint16_t *o = (uint16_t *)ep.out + (int64_t)(m0 + row) * ep.out_sm + n;
        if (ep.wide8 && n + 8 <= n_out) {
            *reinterpret_cast<uint4 *>(o) = v;
        } else {
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (n + k < n_out) o[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
        }
    }
}

// Sums of the splits in their order, then residual or SwiGLU and the one rounding.  Four columns of out per thread.
template <bool GLU>
__global__ __launch_bounds__(256) void join_splits_kernel(const float *__restrict__ partial, int splits, Epilogue ep, int M, int N, int n_tiles) {
    const int cols = GLU ? N / 2 : N, per_row = (cols + 3) / 4;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t m = i / per_row, width = 16LL * n_tiles;
    if (m >= M) return;
    const int n = (int)(i - m * per_row) * 4, at = GLU ? (n >> 3) * 16 + (n & 7) : n;
    const float *p = partial + m * width + at;
    f32x4 y = {0.f, 0.f, 0.f, 0.f}, up = y;
    for (int s = 0; s < splits; ++s, p += (int64_t)M * width) {
        y += *reinterpret_cast<const f32x4 *>(p);
        if constexpr (GLU) up += *reinterpret_cast<const f32x4 *>(p + 8);
    }
    if constexpr (GLU) {
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = ha_silu(y[k]) * up[k];
    }
    if (ep.out_dtype == HA_F32) {
        store4(ep, m, n, cols, y);
        return;
    }
    if (ep.res) add_residual(ep, m, n, cols, y);
    const uint2 v = narrow4(y, ep.out_dtype);
    uint16_t *o = (uint16_t *)ep.out + m * ep.out_sm + n;
    if (ep.wide && n + 4 <= cols) {
        *reinterpret_cast<uint2 *>(o) = v;
    } else {
        const uint32_t w[2] = {v.x, v.y};
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n + k < cols) o[k] = (uint16_t)(w[k >> 1] >> (16 * (k & 1)));
    }
}

struct Args {
    hipStream_t stream;
    const uint8_t *x;
    int64_t x_sm;
    const float *xs;
    int64_t xs_sm;
    const uint8_t *tiles;
    const float *ws;
    Epilogue ep;
    int M, N, act;
    Packed p;
};

// One workgroup per CU, the tiles in equal rounds, workgroups in whole runs of 8 (the XCDs) per group of rows.  Two workgroups per CU,
// where registers allow it, bring nothing: 16 rows, 28672 x 4096 24.3 us against 22.6; 128 rows, 6144 x 1024 8.6 against 7.4.
template <int NWAVE, int KW, int PF, int MT, bool WIDE, bool EXACT>
void launch_rows(const Args &a) {
    const int groups = (a.M + 16 * MT - 1) / (16 * MT);
    const int most = groups <= 32 ? 256 / groups / 8 * 8 : 8, rounds = (a.p.n_tiles + most - 1) / most;
    const unsigned grid = (unsigned)groups * (unsigned)(((a.p.n_tiles + rounds - 1) / rounds + 7) / 8 * 8);
    if (a.act)
        hipLaunchKernelGGL((linear_fp8_rows_kernel<NWAVE, KW, PF, MT, WIDE, EXACT, true>), dim3(grid), dim3(NWAVE * 64), 0, a.stream, a.x,
                           a.x_sm, a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, groups);
    else
        hipLaunchKernelGGL((linear_fp8_rows_kernel<NWAVE, KW, PF, MT, WIDE, EXACT, false>), dim3(grid), dim3(NWAVE * 64), 0, a.stream, a.x,
                           a.x_sm, a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, groups);
}

template <int NWAVE, int PF, int NT, int MT, bool EXACT>
void launch_stream(const Args &a) {
    const int groups = (a.M + 16 * MT - 1) / (16 * MT);
    const unsigned grid = (unsigned)groups * (unsigned)(((a.p.n_tiles + NT - 1) / NT + 7) / 8 * 8);
    if (a.act)
        hipLaunchKernelGGL((linear_fp8_stream_kernel<NWAVE, PF, NT, MT, EXACT, true>), dim3(grid), dim3(NWAVE * 64), 0, a.stream, a.x, a.x_sm,
                           a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, groups);
    else
        hipLaunchKernelGGL((linear_fp8_stream_kernel<NWAVE, PF, NT, MT, EXACT, false>), dim3(grid), dim3(NWAVE * 64), 0, a.stream, a.x, a.x_sm,
                           a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, groups);
}

template <int WN, int WM, int TN, int TM, int AHEAD, bool EXACT>
void launch_tiled(const Args &a) {
    const int tiles_n = (a.p.n_tiles + WN * TN - 1) / (WN * TN), tiles_m = (a.M + 16 * WM * TM - 1) / (16 * WM * TM);
    const int per_xcd = (int)(((int64_t)tiles_n * tiles_m + 7) / 8);
    if (a.act)
        hipLaunchKernelGGL((linear_fp8_tiled_kernel<WN, WM, TN, TM, AHEAD, EXACT, true, false>), dim3(8u * (unsigned)per_xcd), dim3(WN * WM * 64),
                           0, a.stream, a.x, a.x_sm, a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, tiles_n, tiles_m, per_xcd,
                           a.p.kb, nullptr);
    else
        hipLaunchKernelGGL((linear_fp8_tiled_kernel<WN, WM, TN, TM, AHEAD, EXACT, false, false>), dim3(8u * (unsigned)per_xcd), dim3(WN * WM * 64),
                           0, a.stream, a.x, a.x_sm, a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, tiles_n, tiles_m, per_xcd,
                           a.p.kb, nullptr);
}

// Whether x of 17 rows and more stays in registers, weights streamed past it: rows of up to 32 blocks, and at most six tiles for a
// workgroup (N / 16 tiles times M / 64 groups of rows, over 256 workgroups).  Against tiles of 128 x 128, with K cut where
// they are few: 6144 x 4096, 64 rows 11.3 us (15.9), 128 rows 13.2 (19.7), 256 rows 18.7 (23.9); 4096 x 2304, 256 rows 13.4 (18.9),
// 384 rows, six tiles, 19.4 (17.9); 6144 x 2048, 384 rows, nine tiles, 25.7 (18.8).  128 rows and fewer would not fill a tile.
bool keeps_rows(int M, Packed p) { return p.kb <= 32 && (M <= 128 || ((M + 63LL) / 64) * p.n_tiles <= 1536); }

// How many ways K is cut for tiles of 128 x 128: into as many as give every CU a tile, of at least four blocks (cut for two
// tiles per CU instead, the longer sum of the parts costs more than it brings: 4096 x 14336, 256 rows 41 us against 37; not cut 96).
struct Splits {
    int count, per;
};
Splits splits_for(int M, Packed p) {
    if (M <= 16 || keeps_rows(M, p)) return {1, p.kb};
    const int64_t tiles = ((p.n_tiles + 7LL) / 8) * ((M + 127LL) / 128);
    int64_t want = 256 / tiles;
    if (want > p.kb / 4) want = p.kb / 4;
    if (want < 2) return {1, p.kb};
    const int per = (int)((p.kb + want - 1) / want);
    return {(p.kb + per - 1) / per, per};
}

template <bool EXACT>
void launch_split(const Args &a, Splits s, float *partial) {
    const int tiles_n = (a.p.n_tiles + 7) / 8, tiles_m = (a.M + 127) / 128;
    const int per_xcd = (int)(((int64_t)tiles_n * tiles_m * s.count + 7) / 8);
    hipLaunchKernelGGL((linear_fp8_tiled_kernel<2, 2, 4, 4, 1, EXACT, false, true>), dim3(8u * (unsigned)per_xcd), dim3(256), 0, a.stream, a.x,
                       a.x_sm, a.xs, a.xs_sm, a.tiles, a.ws, a.ep, a.M, a.N, a.p.kb, a.p.n_tiles, tiles_n, tiles_m, per_xcd, s.per, partial);
    const int cols = a.act ? a.N / 2 : a.N;
    const unsigned grid = (unsigned)(((int64_t)a.M * ((cols + 3) / 4) + 255) / 256);
    if (a.act)
        hipLaunchKernelGGL(join_splits_kernel<true>, dim3(grid), dim3(256), 0, a.stream, partial, s.count, a.ep, a.M, a.N, a.p.n_tiles);
    else
        hipLaunchKernelGGL(join_splits_kernel<false>, dim3(grid), dim3(256), 0, a.stream, partial, s.count, a.ep, a.M, a.N, a.p.n_tiles);
}

// 17 rows and more, in registers
template <bool EXACT>
void launch_some_rows(const Args &a) {
    if (a.M <= 32) {
        if (a.p.kb <= 8) launch_rows<8, 1, 1, 2, false, EXACT>(a);
        else if (a.p.kb <= 16) launch_rows<8, 2, 2, 2, false, EXACT>(a);
        else launch_rows<8, 4, 4, 2, false, EXACT>(a);
    } else {
        if (a.p.kb <= 8) launch_rows<8, 1, 1, 4, false, EXACT>(a);
        else if (a.p.kb <= 16) launch_rows<8, 2, 2, 4, false, EXACT>(a);
        else launch_rows<8, 4, 2, 4, false, EXACT>(a);
    }
}

}  // namespace

extern "C" {

int64_t ha_weight_fp8_bytes(int N, int K, int glu) {
    if (N < 1 || K < 1 || (glu && N % 2 != 0)) return 0;
    const Packed p = packed_shape(N, K, glu);
    return (int64_t)p.n_tiles * p.kb * kTileBytes;
}

size_t ha_linear_fp8_workspace_bytes(int M, int N, int K, int act) {
    if (M < 1 || ha_weight_fp8_bytes(N, K, act) == 0) return 0;
    const Packed p = packed_shape(N, K, act);
    const Splits s = splits_for(M, p);
    return s.count > 1 ? (size_t)s.count * (size_t)M * 16u * (size_t)p.n_tiles * sizeof(float) : 0;
}

int64_t ha_weight_fp8_scales(int N, int K, int glu) { return ha_weight_fp8_bytes(N, K, glu) / kTileBytes * 2; }

int ha_pack_weight_fp8(const void *w, int64_t w_stride_n, int dtype, const float *w_scales, int64_t w_scales_stride_n, int N, int K, int glu,
                       void *tiles, float *tile_scales, void *stream) {
    HA_REQUIRE(w && tiles && tile_scales, HA_ERR_NULL_POINTER, "w/tiles/tile_scales is NULL");
    HA_REQUIRE(dtype == HA_F32 || dtype == HA_BF16 || dtype == HA_F16 || dtype == HA_FP8_E4M3, HA_ERR_BAD_DTYPE, "unknown dtype %d", dtype);
    HA_REQUIRE((dtype == HA_FP8_E4M3) == (w_scales != nullptr), HA_ERR_NULL_POINTER,
               "weights in e4m3 come with their scales, any other type without");
    HA_REQUIRE(N >= 1 && K >= 1 && K <= HA_FP8_MAX_K && w_stride_n >= K && (glu == 0 || (glu == 1 && N % 2 == 0)), HA_ERR_BAD_SHAPE,
               "need N >= 1, 1 <= K <= %d, an even N for the gate/up form, rows of at least K elements", HA_FP8_MAX_K);
    const Packed p = packed_shape(N, K, glu);
    const int rows = glu ? N / 2 : N, row_blocks = ha_fp8_blocks(rows);
    HA_REQUIRE(!w_scales || w_scales_stride_n >= p.kb, HA_ERR_BAD_SHAPE, "a row of w_scales holds a number for every block of 128 inputs");
    HA_REQUIRE(row_blocks * (glu ? 2LL : 1LL) <= 65535 && ha_fits_launch(p.kb, 256), HA_ERR_BAD_SHAPE, "matrix too large for one launch");
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
                  int out_dtype, int M, int N, int K, void *workspace, size_t workspace_bytes, void *stream) {
    HA_REQUIRE(tiles && tile_scales && (M == 0 || (xq && x_scales && out)), HA_ERR_NULL_POINTER,
               "xq/x_scales/tiles/tile_scales/out is NULL");
    HA_REQUIRE(out_dtype == HA_F32 || out_dtype == HA_BF16 || out_dtype == HA_F16, HA_ERR_BAD_DTYPE, "unknown dtype %d", out_dtype);
    HA_REQUIRE(M >= 0 && N >= 1 && K >= 1 && K <= HA_FP8_MAX_K, HA_ERR_BAD_SHAPE, "need M >= 0, N >= 1, 1 <= K <= %d", HA_FP8_MAX_K);
    HA_REQUIRE(act == HA_ACT_NONE || act == HA_ACT_SWIGLU, HA_ERR_BAD_SHAPE, "unknown activation %d", act);
    HA_REQUIRE(!act || (N % 2 == 0 && !residual), HA_ERR_BAD_SHAPE, "SwiGLU needs an even number of weight rows and no residual");
    const Packed p = packed_shape(N, K, act);
    const int n_out = act ? N / 2 : N;
    HA_REQUIRE(xq_stride_m >= (int64_t)p.kb * HA_FP8_BLOCK && x_scales_stride_m >= p.kb && out_stride_m >= n_out &&
                   (!residual || residual_stride_m == 0 || residual_stride_m >= N),
               HA_ERR_BAD_SHAPE, "strides smaller than the rows they span");
    const int es = ha_dtype_bytes(out_dtype);
    HA_REQUIRE(ha_aligned(xq, 16) && xq_stride_m % 16 == 0 && ha_aligned(tiles, 16), HA_ERR_MISALIGNED,
               "rows of xq and tiles must be 16-byte aligned");
    HA_REQUIRE(ha_aligned(x_scales, 4) && ha_aligned(tile_scales, 8) && ha_aligned(out, es) && ha_aligned(residual, es), HA_ERR_MISALIGNED,
               "pointers are not aligned to their elements");
    int st;
    const bool wide = ha_aligned(out, 4 * es) && out_stride_m % 4 == 0 && (!residual || (ha_aligned(residual, 4 * es) && residual_stride_m % 4 == 0));
    const Epilogue ep = {residual, residual_stride_m, out, out_stride_m, out_dtype, wide, ha_aligned(out, 8 * es) && out_stride_m % 8 == 0};
    const Args a = {(hipStream_t)stream, (const uint8_t *)xq, xq_stride_m, x_scales, x_scales_stride_m, (const uint8_t *)tiles, tile_scales, ep,
                    M, N, act, p};
    const bool exact = out_dtype == HA_F32;
    // offsets within a workgroup's tiles are 32-bit
    const bool in_reach = xq_stride_m < (1LL << 22) && x_scales_stride_m < (1LL << 20) && (int64_t)p.kb * kTileBytes * 16 < (1LL << 31);
    const bool tiled = in_reach && M > 32;
    const int64_t groups = M <= 16 ? p.n_tiles + 7LL
                           : tiled ? ((M + 127LL) / 128) * ((p.n_tiles + 7LL) / 8) + 7
                                   : ((M + 31LL) / 32) * ((p.n_tiles + 1LL) / 2 + 7);
    HA_REQUIRE(ha_fits_launch(groups, M <= 16 ? 1024 : tiled ? 256 : 512), HA_ERR_BAD_SHAPE, "too many tiles for one launch");
    const Splits splits = in_reach ? splits_for(M, p) : Splits{1, p.kb};
    if (splits.count > 1) {
        const size_t need = ha_linear_fp8_workspace_bytes(M, N, K, act);
        HA_REQUIRE(workspace && workspace_bytes >= need, HA_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace_bytes);
        HA_REQUIRE(ha_aligned(workspace, 16), HA_ERR_MISALIGNED, "workspace must be 16-byte aligned");
    }
    st = ha_require_device();
    if (st || M == 0) return st;
    if (splits.count > 1) {
        if (exact) launch_split<true>(a, splits, (float *)workspace);
        else launch_split<false>(a, splits, (float *)workspace);
    } else if (M <= 16) {
        if (p.kb <= 8) launch_rows<8, 1, 1, 1, true, true>(a);
        else if (p.kb <= 16) launch_rows<8, 2, 2, 1, true, true>(a);
        else if (p.kb <= 32) launch_rows<8, 4, 2, 1, true, true>(a);
        else launch_stream<16, 2, 1, 1, true>(a);
    } else if (keeps_rows(M, p)) {
        if (exact) launch_some_rows<true>(a);
        else launch_some_rows<false>(a);
    } else if (tiled) {
        // (up to 32 rows the stream is as fast; 17408 x 4224, 40 rows 29.8 us against the stream's 34.1, 128 rows 36.5 against 66)
        const int64_t big = ((p.n_tiles + 15LL) / 16) * ((M + 255LL) / 256);
        if (exact) launch_tiled<2, 2, 4, 4, 1, true>(a);
        else if (big >= 200) launch_tiled<2, 4, 8, 4, 3, false>(a);
        else launch_tiled<2, 2, 4, 4, 1, false>(a);
    } else {
        if (exact) launch_stream<8, 2, 2, 2, true>(a);
        else launch_stream<8, 2, 2, 2, false>(a);
    }
    HA_CHECK_LAUNCH("ha_linear_fp8");
    return HA_OK;
}

}  // extern "C"
