// wc_linear.hip -- entry points of the products with compressed weights (plain and grouped by expert, forward and the gradient
// of the activations), the kernels that decompress a weight into the workspace of the dense product, and the gradient of the
// epilogue's activation.
//
// The reference answers with a compressed layer by decompressing the whole weight on every read
// (src/nncf/torch/quantization/layers.py:1303-1460) in front of a library product; here the weight is multiplied as stored.
#include "wc_linear.h"

namespace wc {

// k as the dense product takes it: stages of 64, three at least
constexpr int64_t padded(int64_t v) { return v <= 192 ? 192 : (v + 63) / 64 * 64; }

// ---------------------------------------------------------------------------------- weight -> dense rows of the workspace
// [experts * n, kp], kp = k rounded up to 64 (192 at least), the tail zero.  Bound by the bytes (0.5-1 read, 2 written per
// weight).  `lanes` (a power of two) threads follow a row, 8 weights each; a thread takes the same place of kDequantRows rows,
// whose reads are requested together and whose addresses are a scalar apart.  An expert without rows is left out.
// 28672 x 8192 int4: 95 us, 6.2 TB/s; eight NF4 experts of 28672 x 4096, groups of 32: 401 us, 6.1 TB/s.
constexpr int kDequantRows = 4;
template <int MODE, int DT>
__global__ __launch_bounds__(256) void k_dequant_rows(const uint8_t* __restrict__ codes, const void* __restrict__ scale,
                                                      const uint8_t* __restrict__ zp, uint16_t* __restrict__ out, int64_t total_rows,
                                                      int64_t n, uint32_t k, uint32_t kp, uint32_t groups, uint32_t magic_group, int log_lanes,
                                                      const RowMap rows) {
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    fill_nf4<MODE>(lut);
    const uint32_t lanes = 1u << log_lanes, strips = 256u >> log_lanes;  // strips of kDequantRows rows
    const int64_t block0 = (int64_t)blockIdx.x * strips * kDequantRows;
    if (rows.offsets) {  // (a block that reaches into an expert with rows takes all of its rows)
        const int64_t block1 = block0 + strips * kDequantRows < total_rows ? block0 + strips * kDequantRows : total_rows;
        bool any = false;
        for (int64_t e = block0 / n; e <= (block1 - 1) / n; ++e) {
            int64_t lo, hi;
            expert_range(rows, (int)e, lo, hi);
            any = any || lo < hi;
        }
        if (!any) return;
    }
    const uint32_t row_bytes = four_bit(MODE) ? k / 2 : k;
    const uint32_t strip = threadIdx.x >> log_lanes;
    const int64_t row0 = block0 + strip * kDequantRows;
    if (row0 >= total_rows) return;
    const int here = total_rows - row0 < kDequantRows ? (int)(total_rows - row0) : kDequantRows;
    const uint8_t* c0 = codes + row0 * row_bytes;
    const int64_t g0 = row0 * groups;
    uint16_t* o0 = out + row0 * kp;
    for (uint32_t v = threadIdx.x & (lanes - 1); v < kp / 8; v += lanes) {
        if (v * 8 >= k) {
            for (int r = 0; r < here; ++r) *(u32v4*)(o0 + (uint64_t)r * kp + v * 8) = u32v4{0, 0, 0, 0};
            continue;
        }
        const uint32_t g = magic_group ? __umulhi(v, magic_group) : v;
        u32v2 p[kDequantRows];
        uint32_t sc[kDequantRows], zr[kDequantRows];
#pragma unroll
        for (int r = 0; r < kDequantRows; ++r) {
            const uint32_t rr = r < here ? r : 0;
            if constexpr (four_bit(MODE)) p[r].x = *(const uint32_t*)(c0 + (uint64_t)rr * row_bytes + v * 4);
            else p[r] = *(const u32v2*)(c0 + (uint64_t)rr * row_bytes + v * 8);
            const int64_t gi = g0 + rr * groups + g;
            if constexpr (MODE == NNCF_AMD_MXFP4) sc[r] = ((const uint8_t*)scale)[gi];
            else sc[r] = ((const uint16_t*)scale)[gi];
            if constexpr (MODE == NNCF_AMD_INT4_ASYM) zr[r] = (uint32_t)(zp[gi >> 1] >> (4 * (gi & 1))) & 15u;
            if constexpr (MODE == NNCF_AMD_INT8_ASYM) zr[r] = zp[gi];
        }
#pragma unroll
        for (int r = 0; r < kDequantRows; ++r)
            if (r < here) *(u32v4*)(o0 + (uint64_t)r * kp + v * 8) = dequant8<MODE, DT>(p[r].x, p[r].y, par_of<MODE>(sc[r], zr[r]), lut);
    }
}

// any shape: a thread per weight
template <int MODE, int DT>
__global__ __launch_bounds__(256) void k_dequant_rows_any(const uint8_t* __restrict__ codes, const void* __restrict__ scale,
                                                          const uint8_t* __restrict__ zp, uint16_t* __restrict__ out, int64_t total,
                                                          int64_t n, int64_t k, int64_t kp, int64_t gs, const RowMap rows) {
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    fill_nf4<MODE>(lut);
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t row = i / kp, c = i - row * kp;
    if (rows.offsets) {
        int64_t lo, hi;
        expert_range(rows, (int)(row / n), lo, hi);
        if (lo >= hi) return;
    }
    uint16_t w = 0;
    if (c < k) w = dequant1<MODE, DT>(codes, row * k + c, group_par<MODE>(scale, zp, (row * k + c) / gs), lut);
    out[i] = w;
}

// ------------------------------------------------------------------------- weight -> its transpose, for the gradient of x
// [experts, k, np], np = n rounded up to 64 (192 at least), the tail zero: tiles of 64 x 64 turned round in LDS as pairs of
// neighbouring n (rows padded by 4 bytes so that the columns that are written fall on different banks).  Bound by the bytes:
// eight int4 weights of 4096 x 14336 in 290 us, 4.1 TB/s (one tile at a time 340: its reads of 32 bytes a row wait alone).
constexpr int kTurns = 4;
template <int MODE, int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void k_dequant_transposed(const uint8_t* __restrict__ codes, const void* __restrict__ scale,
                                                            const uint8_t* __restrict__ zp, uint16_t* __restrict__ out, int64_t n,
                                                            int64_t k, int64_t np, int64_t gs, const RowMap rows) {
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    __shared__ uint32_t tile[64][33];  // [k][pairs of n]
    fill_nf4<MODE>(lut);
    const int expert = blockIdx.z;
    if (rows.offsets) {
        int64_t lo, hi;
        expert_range(rows, expert, lo, hi);
        if (lo >= hi) return;
    }
    // kTurns tiles one behind the other along k: their reads, 32 or 64 bytes of a row each, are requested together
    const int64_t n0 = (int64_t)blockIdx.x * 64, kb = (int64_t)blockIdx.y * 64 * kTurns, groups = k / gs;
    const int pair = threadIdx.x >> 3, v = (threadIdx.x & 7) * 8;  // a thread: two rows of W, 8 k of each
    u32v2 p[kTurns][2];
    uint32_t sc[kTurns][2], zr[kTurns][2];
    if constexpr (ALIGNED) {
#pragma unroll
        for (int t = 0; t < kTurns; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                int64_t row = n0 + 2 * pair + h, c = kb + 64 * t + v;  // (rows and k behind the end: any, their place gets zeros)
                row = row < n ? row : n - 1;
                c = c < k ? c : 0;
                const int64_t at = (int64_t)expert * n + row, e0 = at * k + c, g = at * groups + (uint32_t)c / (uint32_t)gs;
                if constexpr (four_bit(MODE)) p[t][h].x = *(const uint32_t*)(codes + e0 / 2);
                else p[t][h] = *(const u32v2*)(codes + e0);
                if constexpr (MODE == NNCF_AMD_MXFP4) sc[t][h] = ((const uint8_t*)scale)[g];
                else sc[t][h] = ((const uint16_t*)scale)[g];
                if constexpr (MODE == NNCF_AMD_INT4_ASYM) zr[t][h] = (uint32_t)(zp[g >> 1] >> (4 * (g & 1))) & 15u;
                if constexpr (MODE == NNCF_AMD_INT8_ASYM) zr[t][h] = zp[g];
            }
    }
#pragma unroll
    for (int t = 0; t < kTurns; ++t) {
        const int64_t k0 = kb + 64 * t;
        if (k0 >= k) break;
        uint16_t w[2][8] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = n0 + 2 * pair + h, c = k0 + v;
            if (row >= n) continue;
            if constexpr (ALIGNED) {
                if (c < k) {
                    const u32v4 o = dequant8<MODE, DT>(p[t][h].x, p[t][h].y, par_of<MODE>(sc[t][h], zr[t][h]), lut);
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[h][2 * j] = (uint16_t)o[j], w[h][2 * j + 1] = (uint16_t)(o[j] >> 16);
                }
            } else {
                const int64_t e0 = ((int64_t)expert * n + row) * k + c;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < k) w[h][j] = dequant1<MODE, DT>(codes, e0 + j, group_par<MODE>(scale, zp, (e0 + j) / gs), lut);
            }
        }
        if (t > 0) __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[v + j][pair] = w[0][j] | (uint32_t)w[1][j] << 16;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 2; ++u) {  // 64 rows of k x 8 vectors of 8 n
            const int kr = pair + 32 * u, nv = (threadIdx.x & 7) * 4;
            if (k0 + kr < k && n0 + 2 * nv < np)
                *(u32v4*)(out + ((int64_t)expert * k + k0 + kr) * np + n0 + 2 * nv) =
                    u32v4{tile[kr][nv], tile[kr][nv + 1], tile[kr][nv + 2], tile[kr][nv + 3]};
        }
    }
}

// ---------------------------------------------------------------------- rows of x -> aligned rows, the tail of each zero
__global__ __launch_bounds__(256) void k_pack_rows(const uint16_t* __restrict__ x, int64_t ldx, int64_t k, int64_t kp,
                                                   uint16_t* __restrict__ out, const RowMap rows) {
    const int64_t row = blockIdx.x;
    const uint16_t* src = x + source_row(rows, row) * ldx;
    for (int64_t c = threadIdx.x; c < kp; c += 256) out[row * kp + c] = c < k ? src[c] : (uint16_t)0;
}

// ------------------------------------------------------------------------------------- gradient of the epilogue's activation
// dz = dy * slope (swiglu: both halves), written with row stride ldz and zeros behind n; and the sums of dz's fp32 values
// over chunks of 32 rows, which k_sum_chunks adds up in order (no atomics: the result does not depend on the schedule).
// dz is rounded to the activations' type because the product that takes it reads 16-bit operands.
// A thread takes VEC consecutive columns; the chunk's rows are dealt to 4 waves whose sums meet in LDS, wave 0 first.  Bound by
// the bytes, 8 an element: 2047 x 4096 in 15 us.
constexpr int kChunkRows = 32;
template <int DT, int VEC>
__global__ __launch_bounds__(256) void k_activation_grad(const uint16_t* __restrict__ dy, int64_t ldd, const float* __restrict__ slope,
                                                         int64_t m, int64_t n, int act, uint16_t* __restrict__ dz, int64_t ldz,
                                                         float* __restrict__ sums) {
    __shared__ float part[3][2 * VEC][64];
    const int64_t width = act == kActSwiglu ? n / 2 : n;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + lane) * VEC;
    const int64_t r0 = (int64_t)blockIdx.y * kChunkRows, r1 = r0 + kChunkRows < m ? r0 + kChunkRows : m;
    float s0[VEC], s1[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) s0[i] = s1[i] = 0.0f;
    auto read = [&](const uint16_t* p, float* v) {
        if constexpr (VEC == 4) {
            const u32v2 w = *(const u32v2*)p;
            v[0] = to_f32<DT>((uint16_t)w.x), v[1] = to_f32<DT>((uint16_t)(w.x >> 16));
            v[2] = to_f32<DT>((uint16_t)w.y), v[3] = to_f32<DT>((uint16_t)(w.y >> 16));
        } else {
            v[0] = to_f32<DT>(*p);
        }
    };
    auto read32 = [&](const float* p, float* v) {
        if constexpr (VEC == 4) {
            const f32x4 w = *(const f32x4*)p;
            v[0] = w.x, v[1] = w.y, v[2] = w.z, v[3] = w.w;
        } else {
            v[0] = *p;
        }
    };
    auto write = [&](uint16_t* p, const float* v) {
        if constexpr (VEC == 4) *(u32v2*)p = u32v2{pair_of<DT>(v[0], v[1]), pair_of<DT>(v[2], v[3])};
        else *p = from_f32<DT>(v[0]);
    };
    if (c < width) {
#pragma unroll 2
        for (int64_t r = r0 + wave; r < r1; r += 4) {
            float g[VEC], a[VEC];
            read(dy + r * ldd + c, g);
            if (act == kActSwiglu) {
                float sg[VEC], su[VEC], b[VEC];
                read32(slope + r * n + c, sg);
                read32(slope + r * n + width + c, su);
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    a[i] = g[i] * sg[i];
                    b[i] = g[i] * su[i];
                    s1[i] += b[i];
                }
                if (dz) write(dz + r * ldz + width + c, b);
            } else if (act != kActNone) {
                float v[VEC];
                read32(slope + r * n + c, v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) a[i] = g[i] * v[i];
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i) a[i] = g[i];
            }
#pragma unroll
            for (int i = 0; i < VEC; ++i) s0[i] += a[i];
            if (dz) write(dz + r * ldz + c, a);
        }
    } else if (dz) {  // the padding's columns, by the threads behind the last column
        for (int i = 0; i < VEC; ++i) {
            const int64_t pad = n + (c - width) + i;
            if (pad < ldz)
                for (int64_t r = r0 + wave; r < r1; r += 4) dz[r * ldz + pad] = 0;
        }
    }
    if (!sums) return;
    if (wave > 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) part[wave - 1][i][lane] = s0[i], part[wave - 1][VEC + i][lane] = s1[i];
    }
    __syncthreads();
    if (wave == 0 && c < width) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            for (int w = 0; w < 3; ++w) s0[i] += part[w][i][lane], s1[i] += part[w][VEC + i][lane];
            sums[blockIdx.y * n + c + i] = s0[i];
            if (act == kActSwiglu) sums[blockIdx.y * n + width + c + i] = s1[i];
        }
    }
}

// a wave of 64 columns; the chunks in four parts, one per wave, joined in order
template <int DT>
__global__ __launch_bounds__(256) void k_sum_chunks(const float* __restrict__ sums, int64_t chunks, int64_t n, uint16_t* __restrict__ out) {
    __shared__ float part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane, per = (chunks + 3) / 4;
    const int64_t i1 = (wave + 1) * per < chunks ? (wave + 1) * per : chunks;
    float s = 0.0f;
    if (c < n) {
#pragma unroll 8
        for (int64_t i = wave * per; i < i1; ++i) s += sums[i * n + c];
    }
    part[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < n) out[c] = from_f32<DT>(part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane]);
}

// ------------------------------------------------------------------------------------------------------------------- host
struct Weight {
    const uint8_t* codes;
    const void* scale;
    const uint8_t* zp;
    int mode;
    int64_t n, k, gs, experts;
};

bool aligned_groups(const Weight& w) {  // 8 consecutive weights of a row: one group, one aligned load
    return w.k % 8 == 0 && w.gs % 8 == 0 && w.k <= 131072 && ((uintptr_t)w.codes & 7) == 0;
}

template <int DT>
int dequant_rows(const Weight& w, const RowMap& rows, uint16_t* out, hipStream_t s) {
    const int64_t kp = padded(w.k), total_rows = w.experts * w.n, groups = w.k / w.gs;
    const bool fast = aligned_groups(w);
    int log_lanes = 3;
    while (log_lanes < 8 && (8ll << log_lanes) < kp) ++log_lanes;
    const int64_t per_block = (256 >> log_lanes) * kDequantRows;
    const int64_t blocks = fast ? (total_rows + per_block - 1) / per_block : (total_rows * kp + 255) / 256;
    if (blocks > 0x7fffffff) {
        set_error("linear: weight too large");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    // ceil(2^32 / (vectors of a group)): exact below 2^14 vectors; 0 for groups of one vector
    const uint32_t per_group = (uint32_t)(w.gs / 8);
    const uint32_t magic = fast && per_group > 1 ? (uint32_t)((((uint64_t)1 << 32) + per_group - 1) / per_group) : 0;
#define GO(M)                                                                                                                  \
    if (fast)                                                                                                                  \
        hipLaunchKernelGGL((k_dequant_rows<M, DT>), dim3((unsigned)blocks), dim3(256), 0, s, w.codes, w.scale, w.zp, out, total_rows, \
                           w.n, (uint32_t)w.k, (uint32_t)kp, (uint32_t)groups, magic, log_lanes, rows);                       \
    else                                                                                                                       \
        hipLaunchKernelGGL((k_dequant_rows_any<M, DT>), dim3((unsigned)blocks), dim3(256), 0, s, w.codes, w.scale, w.zp, out,  \
                           total_rows * kp, w.n, w.k, kp, w.gs, rows);
#define BY_MODE                                                          \
    switch (w.mode) {                                                    \
        case NNCF_AMD_INT8_ASYM: GO(NNCF_AMD_INT8_ASYM) break;           \
        case NNCF_AMD_INT8_SYM: GO(NNCF_AMD_INT8_SYM) break;             \
        case NNCF_AMD_INT4_ASYM: GO(NNCF_AMD_INT4_ASYM) break;           \
        case NNCF_AMD_INT4_SYM: GO(NNCF_AMD_INT4_SYM) break;             \
        case NNCF_AMD_NF4: GO(NNCF_AMD_NF4) break;                       \
        default: GO(NNCF_AMD_MXFP4) break;                               \
    }
    BY_MODE
#undef GO
    return launch_status("linear: decompression");
}

template <int DT>
int dequant_transposed(const Weight& w, const RowMap& rows, uint16_t* out, hipStream_t s) {
    const int64_t np = padded(w.n), tn = np / 64, tk = (w.k + 64 * kTurns - 1) / (64 * kTurns);
    if (tn > 0x7fffffff || tk > 65535 || w.experts > 65535) {
        set_error("linear: weight too large");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    const dim3 grid((unsigned)tn, (unsigned)tk, (unsigned)w.experts);
    const bool fast = aligned_groups(w);
#define GO(M)                                                                                                                    \
    if (fast)                                                                                                                    \
        hipLaunchKernelGGL((k_dequant_transposed<M, DT, true>), grid, dim3(256), 0, s, w.codes, w.scale, w.zp, out, w.n, w.k, np, w.gs, rows); \
    else                                                                                                                         \
        hipLaunchKernelGGL((k_dequant_transposed<M, DT, false>), grid, dim3(256), 0, s, w.codes, w.scale, w.zp, out, w.n, w.k, np, w.gs, rows);
    BY_MODE
#undef GO
#undef BY_MODE
    return launch_status("linear: decompression");
}

int check_weight(const char* what, int dtype, const Weight& w) {
    if (dtype != NNCF_AMD_F16 && dtype != NNCF_AMD_BF16) {
        set_error("%s: activations are fp16 or bf16 (dtype %d)", what, dtype);
        return NNCF_AMD_ERR_DTYPE;
    }
    if (w.mode < NNCF_AMD_INT8_ASYM || w.mode > NNCF_AMD_MXFP4) {
        set_error("%s: unsupported mode %d", what, w.mode);
        return NNCF_AMD_ERR_MODE;
    }
    if (w.n < 1 || w.k < 1 || w.experts < 1) {
        set_error("%s: bad shape (n=%lld k=%lld experts=%lld)", what, (long long)w.n, (long long)w.k, (long long)w.experts);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (w.gs < 1 || w.k % w.gs) {
        set_error("Channel size %lld should be divisible by size of group %lld.", (long long)w.k, (long long)w.gs);
        return NNCF_AMD_ERR_GROUP_SIZE;
    }
    if (four_bit(w.mode) && (w.experts * w.n * w.k) % 2) {
        set_error("%s: 4-bit weight with an odd number of elements", what);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (w.experts > (1 << 20) || w.n > ((int64_t)1 << 31) || w.k > ((int64_t)1 << 31)) {
        set_error("%s: shape beyond the kernels' range", what);
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    return NNCF_AMD_OK;
}
int check_pointers(const char* what, const Weight& w) {
    if (!w.codes || !w.scale) {
        set_error("%s: null weight", what);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if ((w.mode == NNCF_AMD_INT8_ASYM || w.mode == NNCF_AMD_INT4_ASYM) && !w.zp) {
        set_error("%s: asymmetric mode needs the zero points", what);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    return NNCF_AMD_OK;
}

// What a call's workspace holds, one behind the other: the decompressed weight, the packed rows of x; and whether the product
// runs on the codes themselves, by strips for few rows (`few`) or by tiles (`tiles`): whichever way's estimate is the least.
struct Need {
    size_t weight, pack;  // (the codes' product: the sums of blocks that share k in the weight's place)
    bool few, tiles;
    FewShape shape;
    CodesShape codes;
    size_t total() const { return weight + pack; }
};
// The time of the dense way in us: the weight decompressed (2.6 bytes an element at 6 TB/s; 8-bit codes take 3) and multiplied by
// 128 x 128 or 256 x 256 tiles (1 and 1.6 us for 64 k of a round of blocks, the former 0.6 where half the blocks fill it).
// Device time in us by strips, tiles and densely, all on one card, the quickest chosen but where noted:
//   28672 x 8192      64 rows           128 rows           256 rows           512 rows           1024 rows
//   int4, groups 128  80 110 240        152 112 240        289 145 267        549 310 325        1070 588 520
//   int4 asymmetric   85 117 295        167 118 270        302 150 272        608 309 318        1130 620 503
//   NF4, groups 64    89 117 249        167 116 275        311 154 276        603 316 314        1182 624 508
//   mxfp4             77 87 258         134 91 276         244 132 269        477 265 336        934 540 491
//   int8              77 105 257 (*)    153 112 266        312 200 288        645 424 336        1219 767 520
//   Eight int4 experts of 4096 x 14336: 436, 322, 538 for 1200 rows; 631, 437, 591 for 2000; 828, 543, 618 for 3000; 1617, 1057,
//   926 for 6000.
// Over these five modes and asymmetric int8, 4096 x 4096 and 4096 x 14336 beside this weight, and twelve numbers of rows from 16 to
// 2048, the choice is within 14 % of the quickest but (*) at 48 and 64 rows: tiles are taken where strips are 21 to 37 % quicker for
// 8-bit codes, and strips where tiles are 18 to 20 % (NF4) and 64 % (mxfp4) quicker on 4096 x 14336.
double dense_us(const Weight& w, int64_t rows, bool grouped) {
    auto blocks = [&](int64_t tile) { return ((w.n + tile - 1) / tile) * ((rows + tile - 1) / tile + (grouped ? (w.experts - 1) / 2 : 0)); };
    const int64_t small = blocks(128), large = blocks(256), steps = (w.k + 63) / 64;
    const double t128 = small <= 256 ? 0.6 : (double)((small + 511) / 512), t256 = 1.6 * (double)((large + 255) / 256);
    return (double)w.experts * (double)w.n * (double)w.k * 2.6 / 6.0e6 + (double)steps * (t128 < t256 ? t128 : t256) + 8.0;
}
bool must_pack(const void* x, int64_t ldx, int64_t k, int64_t sources, bool gathered) {
    return k != padded(k) || ldx % 8 || ((uintptr_t)x & 15) || !dense_reaches(1, 32, ldx, sources, false, gathered);
}
Need forward_need(const Weight& w, const void* x, int64_t ldx, int64_t sources, bool gathered, int64_t rows, bool gated, bool grouped) {
    Need d{(size_t)(w.experts * w.n * padded(w.k)) * 2, 0, false, false, {}, {}};
    const bool copy = ldx % 8 || ((uintptr_t)x & 15);
    d.few = rows <= 1024 * w.experts && few_fits(w.mode, w.k, w.gs, w.codes, copy ? rows : sources, copy ? padded(w.k) : ldx);
    double us = dense_us(w, rows, grouped);
    if (d.few) {
        d.shape = few_plan(w.mode, w.n, w.k, w.k / w.gs, gated, rows, w.experts, grouped);
        d.few = (double)d.shape.cost * 0.12 < us;
        if (d.few) us = (double)d.shape.cost * 0.12;
    }
    // (tiles are not asked where strips win by far: a search of a microsecond in calls of ten)
    if ((!d.few || rows > 32 * w.experts) && rows <= 4096 * w.experts && w.k == padded(w.k) && codes_fits(w.mode, w.n, w.k, w.gs, w.codes)) {
        d.codes = codes_plan(w.mode, w.n, w.k, gated, rows, w.experts, grouped);
        d.tiles = d.codes.us < us;
        if (d.tiles) d.few = false;
    }
    const int kz = d.few ? d.shape.kz : d.tiles ? d.codes.kz : 0;
    if (kz) d.weight = kz > 1 ? (size_t)(kz * rows * w.n + 3) / 4 * 16 : 0;
    if (d.few ? copy : must_pack(x, ldx, w.k, sources, gathered)) d.pack = (size_t)(rows * padded(w.k)) * 2;
    return d;
}
Need backward_need(const Weight& w, const void* dz, int64_t ldz, int64_t rows) {
    Need d{(size_t)(w.experts * w.k * padded(w.n)) * 2, 0, false, false, {}, {}};
    if (must_pack(dz, ldz, w.n, rows, false)) d.pack = (size_t)(rows * padded(w.n)) * 2;
    return d;
}

int vec_of(const Epilogue& e) {
    const int64_t width = e.act == kActSwiglu ? e.n / 2 : e.n;
    uintptr_t bits = (uintptr_t)e.y | (uintptr_t)e.residual;
    if (e.y32 && ((uintptr_t)e.y & 15)) return 0;
    return (bits & 7) == 0 && ((uintptr_t)e.slope & 15) == 0 && e.ldy % 4 == 0 && (!e.residual || e.ldr % 4 == 0) && (!e.slope || width % 4 == 0);
}

int pack_rows(const void*& x, int64_t& ldx, int64_t k, RowMap& rows, uint16_t* pack, hipStream_t s) {
    const int64_t kp = padded(k);
    if (rows.rows > 0x7fffffff) {
        set_error("linear: too many rows");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    hipLaunchKernelGGL(k_pack_rows, dim3((unsigned)rows.rows), dim3(256), 0, s, (const uint16_t*)x, ldx, k, kp, pack, rows);
    x = pack, ldx = kp, rows.slots = nullptr, rows.sources = rows.rows;
    return launch_status("linear: rows");
}

int lds_refused(int bytes) {
    (void)hipGetLastError();  // (reported here, not by the next launch)
    set_error("linear: %d bytes of LDS refused", bytes);
    return NNCF_AMD_ERR_LAUNCH;
}

int out_of_range(int64_t n, int64_t k) {
    set_error("linear: operands beyond the kernels' range (n=%lld k=%lld)", (long long)n, (long long)k);
    return NNCF_AMD_ERR_UNSUPPORTED;
}

int run_dense(int dtype, const void* x, int64_t ldx, int64_t k, const void* w, RowMap rows, Epilogue ep, uint16_t* pack, hipStream_t s) {
    const int64_t kp = padded(k);
    if (must_pack(x, ldx, k, rows.sources, rows.slots != nullptr)) {
        const int st = pack_rows(x, ldx, k, rows, pack, s);
        if (st != NNCF_AMD_OK) return st;
    }
    if (!dense_reaches(ep.n, kp, ldx, rows.sources, ep.act == kActSwiglu, rows.slots != nullptr)) return out_of_range(ep.n, k);
    ep.vec = vec_of(ep);
    return dense_launch(dtype, DenseArgs{x, w, ldx, kp, rows, ep}, s);
}

int forward(const char* what, const void* x, int dtype, int64_t ldx, const Weight& w, const RowMap& rows, const Epilogue& ep, void* ws,
            size_t ws_bytes, hipStream_t s) {
    if (ep.act < kActNone || ep.act > kActSwiglu) {
        set_error("%s: unknown activation %d", what, ep.act);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (ep.act == kActSwiglu && w.n % 2) {
        set_error("%s: swiglu needs an even number of weight rows (n=%lld)", what, (long long)w.n);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const int64_t width = ep.act == kActSwiglu ? w.n / 2 : w.n;
    if (rows.rows == 0) return NNCF_AMD_OK;
    int st = check_pointers(what, w);
    if (st != NNCF_AMD_OK) return st;
    if (!x || !ep.y || ldx < w.k || ep.ldy < width || (ep.residual && ep.ldr < width)) {
        set_error("%s: null or overlapping rows (ldx=%lld ldy=%lld)", what, (long long)ldx, (long long)ep.ldy);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const Need need = forward_need(w, x, ldx, rows.sources, rows.slots != nullptr, rows.rows, ep.act == kActSwiglu, rows.offsets != nullptr);
    if (need.total() && (!ws || ws_bytes < need.total() || ((uintptr_t)ws & 15))) {
        set_error("%s: workspace of %zu bytes, aligned to 16, needed", what, need.total());
        return NNCF_AMD_ERR_WORKSPACE;
    }
    if (need.few) {
        RowMap map = rows;
        if (need.pack) {
            st = pack_rows(x, ldx, w.k, map, (uint16_t*)((char*)ws + need.weight), s);
            if (st != NNCF_AMD_OK) return st;
        }
        const uint32_t g16 = (uint32_t)(w.gs / 16);  // at least 2: groups of whole 32
        const uint32_t magic = (uint32_t)((((uint64_t)1 << 32) + g16 - 1) / g16);
        const uint32_t groups = (uint32_t)(w.k / w.gs);
        // (more than eight groups, so that the multiplier fits; their number times 16 rows of 8 strips stays far below 2^32)
        const bool eights = groups % 8 == 0 && groups > 8 && (((uintptr_t)w.scale | (uintptr_t)w.zp) & 15) == 0;
        const uint32_t scales8 = eights ? (uint32_t)((((uint64_t)1 << 32) + groups / 8 - 1) / (groups / 8)) : 0;
        Epilogue e = ep;
        e.vec = vec_of(e);
        return few_launch(dtype, w.mode, FewArgs{x, ldx, w.codes, w.scale, w.zp, (uint32_t)w.k, groups, magic, scales8, map, e, (float*)ws}, need.shape, s);
    }
    if (need.tiles) {
        RowMap map = rows;
        if (need.pack) {
            st = pack_rows(x, ldx, w.k, map, (uint16_t*)((char*)ws + need.weight), s);
            if (st != NNCF_AMD_OK) return st;
        }
        if (!dense_reaches(w.n, w.k, ldx, map.sources, ep.act == kActSwiglu, map.slots != nullptr)) return out_of_range(w.n, w.k);
        const uint32_t stages = w.gs % 64 ? 0 : (uint32_t)(w.gs / 64);
        const uint64_t magic = stages ? (((uint64_t)1 << 32) + stages - 1) / stages : 0;
        Epilogue e = ep;
        e.vec = vec_of(e);
        return codes_launch(dtype, w.mode, need.codes.fb,
                            CodesArgs{x, ldx, w.k, w.codes, w.scale, w.zp, (uint32_t)(w.k / w.gs), stages, magic, map, e, (float*)ws, need.codes.kz}, s);
    }
    uint16_t* dense = (uint16_t*)ws;
    st = dtype == NNCF_AMD_BF16 ? dequant_rows<NNCF_AMD_BF16>(w, rows, dense, s) : dequant_rows<NNCF_AMD_F16>(w, rows, dense, s);
    if (st != NNCF_AMD_OK) return st;
    return run_dense(dtype, x, ldx, w.k, dense, rows, ep, (uint16_t*)((char*)ws + need.weight), s);
}

int backward(const char* what, const void* dz, int dtype, int64_t ldz, const Weight& w, const RowMap& rows, void* dx, int64_t ldx,
             int dx32, void* ws, size_t ws_bytes, hipStream_t s) {
    if (rows.rows == 0) return NNCF_AMD_OK;
    int st = check_pointers(what, w);
    if (st != NNCF_AMD_OK) return st;
    if (!dz || !dx || ldz < w.n || ldx < w.k) {
        set_error("%s: null or overlapping rows (ldz=%lld ldx=%lld)", what, (long long)ldz, (long long)ldx);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const Need need = backward_need(w, dz, ldz, rows.rows);
    if (!ws || ws_bytes < need.total() || ((uintptr_t)ws & 15)) {
        set_error("%s: workspace of %zu bytes, aligned to 16, needed", what, need.total());
        return NNCF_AMD_ERR_WORKSPACE;
    }
    uint16_t* dense = (uint16_t*)ws;
    st = dtype == NNCF_AMD_BF16 ? dequant_transposed<NNCF_AMD_BF16>(w, rows, dense, s) : dequant_transposed<NNCF_AMD_F16>(w, rows, dense, s);
    if (st != NNCF_AMD_OK) return st;
    Epilogue ep{};
    ep.y = dx, ep.ldy = ldx, ep.n = w.k, ep.y32 = dx32;
    return run_dense(dtype, dz, ldz, w.n, dense, rows, ep, (uint16_t*)((char*)ws + need.weight), s);
}

int check_groups(const char* what, const int32_t* offsets, const int32_t* slots, int64_t topk, int64_t rows, int64_t sources) {
    if (rows < 0 || rows > 0x7fffffff || sources < 0 || topk < 1 || topk > 0x7fffffff) {
        set_error("%s: bad shape (rows=%lld sources=%lld topk=%lld)", what, (long long)rows, (long long)sources, (long long)topk);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (rows > 0 && (!offsets || sources < 1 || (!slots && sources != rows))) {
        set_error("%s: null offsets, or rows without their sources", what);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    return NNCF_AMD_OK;
}

}  // namespace wc

extern "C" size_t nncf_amd_compressed_linear_workspace(const void* x, int64_t ldx, int64_t m, int64_t n, int64_t k, const void* codes,
                                                       int mode, int64_t group_size, int activation) {
    using namespace wc;
    if (m < 1 || n < 1 || k < 1) return 0;
    const Weight w{(const uint8_t*)codes, nullptr, nullptr, mode, n, k, group_size == -1 ? k : group_size, 1};
    if (w.gs < 1 || k % w.gs) return 0;  // (the call refuses it)
    return forward_need(w, x, ldx, m, false, m, activation == kActSwiglu, false).total();
}

extern "C" int nncf_amd_compressed_linear(const void* x, int dtype, int64_t ldx, int64_t m, int64_t n, int64_t k, const void* codes, int mode,
                                          int64_t group_size, const void* scale, const uint8_t* zero_point, const void* bias, int activation,
                                          const void* residual, int64_t ldr, void* y, int64_t ldy, float* slope, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    using namespace wc;
    const Weight w{(const uint8_t*)codes, scale, zero_point, mode, n, k, group_size == -1 ? k : group_size, 1};
    const int st = check_weight("compressed_linear", dtype, w);
    if (st != NNCF_AMD_OK) return st;
    if (m < 0 || m > 0x7fffffff) {
        set_error("compressed_linear: bad number of rows %lld", (long long)m);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const RowMap rows{nullptr, nullptr, 1, 1, m, m};
    Epilogue ep{};
    ep.bias = bias, ep.residual = residual, ep.y = y, ep.slope = slope, ep.ldr = ldr, ep.ldy = ldy, ep.n = n, ep.act = activation;
    return forward("compressed_linear", x, dtype, ldx, w, rows, ep, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" size_t nncf_amd_expert_linear_workspace(const void* x, int64_t ldx, int64_t sources, int gathered, int64_t rows, int64_t n,
                                                   int64_t k, const void* codes, int mode, int64_t group_size, int64_t experts, int activation) {
    using namespace wc;
    if (rows < 1 || n < 1 || k < 1 || experts < 1) return 0;
    const Weight w{(const uint8_t*)codes, nullptr, nullptr, mode, n, k, group_size == -1 ? k : group_size, experts};
    if (w.gs < 1 || k % w.gs) return 0;  // (the call refuses it)
    return forward_need(w, x, ldx, sources, gathered != 0, rows, activation == kActSwiglu, true).total();
}

extern "C" int nncf_amd_expert_linear(const void* x, int dtype, int64_t ldx, int64_t sources, const int32_t* slots, int64_t topk,
                                      const int32_t* offsets, int64_t experts, int64_t rows, int64_t n, int64_t k, const void* codes,
                                      int mode, int64_t group_size, const void* scale, const uint8_t* zero_point, int activation, void* y,
                                      int64_t ldy, float* slope, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace wc;
    const Weight w{(const uint8_t*)codes, scale, zero_point, mode, n, k, group_size == -1 ? k : group_size, experts};
    int st = check_weight("expert_linear", dtype, w);
    if (st == NNCF_AMD_OK) st = check_groups("expert_linear", offsets, slots, topk, rows, sources);
    if (st != NNCF_AMD_OK) return st;
    const RowMap map{offsets, slots, (int32_t)experts, (int32_t)topk, rows, sources};
    Epilogue ep{};
    ep.y = y, ep.slope = slope, ep.ldy = ldy, ep.n = n, ep.act = activation;
    return forward("expert_linear", x, dtype, ldx, w, map, ep, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" size_t nncf_amd_linear_grad_input_workspace(const void* dz, int64_t ldz, int64_t rows, int64_t n, int64_t k, int64_t experts) {
    using namespace wc;
    if (rows < 1 || n < 1 || k < 1 || experts < 1) return 0;
    const Weight w{nullptr, nullptr, nullptr, 0, n, k, k, experts};
    return backward_need(w, dz, ldz, rows).total();
}

extern "C" int nncf_amd_linear_grad_input(const void* dz, int dtype, int64_t ldz, const int32_t* offsets, int64_t experts, int64_t rows,
                                          int64_t n, int64_t k, const void* codes, int mode, int64_t group_size, const void* scale,
                                          const uint8_t* zero_point, void* dx, int64_t ldx, int dx_is_f32, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    using namespace wc;
    const Weight w{(const uint8_t*)codes, scale, zero_point, mode, n, k, group_size == -1 ? k : group_size, experts};
    const int st = check_weight("linear_grad_input", dtype, w);
    if (st != NNCF_AMD_OK) return st;
    if (rows < 0 || rows > 0x7fffffff || (!offsets && experts != 1)) {
        set_error("linear_grad_input: bad shape (rows=%lld experts=%lld)", (long long)rows, (long long)experts);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const RowMap map{offsets, nullptr, (int32_t)experts, 1, rows, rows};
    return backward("linear_grad_input", dz, dtype, ldz, w, map, dx, ldx, dx_is_f32, workspace, workspace_bytes, (hipStream_t)stream);
}

extern "C" size_t nncf_amd_activation_grad_workspace(int64_t m, int64_t n) {
    return m < 1 || n < 1 ? 0 : (size_t)((m + wc::kChunkRows - 1) / wc::kChunkRows) * (size_t)n * 4;
}

extern "C" int nncf_amd_activation_grad(const void* dy, int dtype, int64_t ldd, const float* slope, int64_t m, int64_t n, int activation, void* dz,
                                        int64_t ldz, void* dbias, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace wc;
    if (dtype != NNCF_AMD_F16 && dtype != NNCF_AMD_BF16) {
        set_error("activation_grad: fp16 or bf16 (dtype %d)", dtype);
        return NNCF_AMD_ERR_DTYPE;
    }
    if (m < 0 || n < 1 || activation < kActNone || activation > kActSwiglu || (activation == kActSwiglu && n % 2)) {
        set_error("activation_grad: bad argument (m=%lld n=%lld activation=%d)", (long long)m, (long long)n, activation);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const int64_t width = activation == kActSwiglu ? n / 2 : n;
    const int64_t chunks = (m + kChunkRows - 1) / kChunkRows;
    // four columns a thread where every row of every operand allows 8-byte accesses
    const bool wide = width % 4 == 0 && n % 4 == 0 && ldd % 4 == 0 && (!dz || ldz % 4 == 0) && (((uintptr_t)dy | (uintptr_t)dz) & 7) == 0 &&
                      ((uintptr_t)slope & 15) == 0;
    const int64_t per = wide ? 256 : 64, blocks = (width + (dz ? ldz - n : 0) + per - 1) / per;
    if (m > 0 && (!dy || ldd < width || (activation != kActNone && !slope) || (dz && ldz < n))) {
        set_error("activation_grad: null or overlapping rows (ldd=%lld ldz=%lld)", (long long)ldd, (long long)ldz);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (blocks > 0x7fffffff) {
        set_error("activation_grad: too many columns");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    if (dbias && m > 0 && (!workspace || workspace_bytes < nncf_amd_activation_grad_workspace(m, n))) {
        set_error("activation_grad: workspace of %zu bytes needed", nncf_amd_activation_grad_workspace(m, n));
        return NNCF_AMD_ERR_WORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    float* sums = dbias ? (float*)workspace : nullptr;
    for (int64_t c0 = 0; c0 < chunks && (dz || dbias); c0 += 65535) {  // the grid's second axis ends at 65535
        const int64_t r0 = c0 * kChunkRows, part = chunks - c0 < 65535 ? chunks - c0 : 65535;
        const int64_t here = m - r0 < part * kChunkRows ? m - r0 : part * kChunkRows;
        const dim3 grid((unsigned)blocks, (unsigned)part);
        const uint16_t* d = (const uint16_t*)dy + r0 * ldd;
        const float* sl = slope ? slope + r0 * n : nullptr;
        uint16_t* z = dz ? (uint16_t*)dz + r0 * ldz : nullptr;
        float* to = sums ? sums + c0 * n : nullptr;
#define GO(DT, VEC) hipLaunchKernelGGL((k_activation_grad<DT, VEC>), grid, dim3(256), 0, s, d, ldd, sl, here, n, activation, z, ldz, to)
        if (dtype == NNCF_AMD_BF16) {
            if (wide) GO(NNCF_AMD_BF16, 4);
            else GO(NNCF_AMD_BF16, 1);
        } else {
            if (wide) GO(NNCF_AMD_F16, 4);
            else GO(NNCF_AMD_F16, 1);
        }
#undef GO
        const int st = launch_status("activation_grad");
        if (st != NNCF_AMD_OK) return st;
    }
    if (dbias) {
        const dim3 grid((unsigned)((n + 63) / 64));
        if (dtype == NNCF_AMD_BF16)
            hipLaunchKernelGGL((k_sum_chunks<NNCF_AMD_BF16>), grid, dim3(256), 0, s, sums, chunks, n, (uint16_t*)dbias);
        else
            hipLaunchKernelGGL((k_sum_chunks<NNCF_AMD_F16>), grid, dim3(256), 0, s, sums, chunks, n, (uint16_t*)dbias);
        return launch_status("activation_grad");
    }
    return NNCF_AMD_OK;
}
