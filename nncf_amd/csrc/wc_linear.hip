// wc_linear.hip -- entry points of the products with compressed weights (plain and grouped by expert, forward and the gradient
// of the activations), the kernels that decompress a weight into the workspace of the dense product, and the gradient of the
// epilogue's activation.
//
// The reference answers with a compressed layer by decompressing the whole weight on every read
// (src/nncf/torch/quantization/layers.py:1303-1460) in front of a library product; here the weight is multiplied as stored.
#include "wc_linear.h"

namespace wc {

constexpr int64_t round64(int64_t v) { return (v + 63) / 64 * 64; }

// ---------------------------------------------------------------------------------- weight -> dense rows of the workspace
// [experts * n, kp], kp = k rounded up to 64, the tail zero.  Bound by the bytes (0.5-1 read, 2 written per weight).  A block
// takes ROWS rows; a thread 8 consecutive weights of a row, whose place and group come from multiplications by 2^32 / d
// (exact while the product of both factors is below 2^32: k up to 131072).  An expert without rows is left out.
constexpr int kDequantRows = 8;
template <int MODE, int DT>
__global__ __launch_bounds__(256) void k_dequant_rows(const uint8_t* __restrict__ codes, const void* __restrict__ scale,
                                                      const uint8_t* __restrict__ zp, uint16_t* __restrict__ out, int64_t total_rows,
                                                      int64_t n, uint32_t k, uint32_t kp, uint32_t groups, uint32_t magic_row,
                                                      uint32_t magic_group, const RowMap rows) {
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    fill_nf4<MODE>(lut);
    const int64_t row0 = (int64_t)blockIdx.x * kDequantRows;
    const uint32_t vecs = kp / 8;
    for (uint32_t i = threadIdx.x; i < kDequantRows * vecs; i += 256) {
        const uint32_t r = __umulhi(i, magic_row), v = i - r * vecs;
        const int64_t row = row0 + r;
        if (row >= total_rows) break;
        if (rows.offsets) {
            int64_t lo, hi;
            expert_range(rows, (int)(row / n), lo, hi);
            if (lo >= hi) continue;
        }
        u32v4 w{0, 0, 0, 0};
        if (v * 8 < k) {
            const GroupPar<MODE> g = group_par<MODE>(scale, zp, row * groups + __umulhi(v, magic_group));
            const int64_t e0 = row * k + v * 8;
            if constexpr (four_bit(MODE)) {
                w = dequant8<MODE, DT>(*(const uint32_t*)(codes + e0 / 2), 0, g, lut);
            } else {
                const u32v2 p = *(const u32v2*)(codes + e0);
                w = dequant8<MODE, DT>(p.x, p.y, g, lut);
            }
        }
        *(u32v4*)(out + row * kp + v * 8) = w;
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
// [experts, k, np], np = n rounded up to 64, the tail zero: tiles of 64 x 64 turned round in LDS (rows padded by 4 bytes so
// that the columns that are written fall on different banks).
template <int MODE, int DT, bool ALIGNED>
__global__ __launch_bounds__(256) void k_dequant_transposed(const uint8_t* __restrict__ codes, const void* __restrict__ scale,
                                                            const uint8_t* __restrict__ zp, uint16_t* __restrict__ out, int64_t n,
                                                            int64_t k, int64_t np, int64_t gs, const RowMap rows) {
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    __shared__ uint16_t tile[64][66];  // [k][n]
    fill_nf4<MODE>(lut);
    const int expert = blockIdx.z;
    if (rows.offsets) {
        int64_t lo, hi;
        expert_range(rows, expert, lo, hi);
        if (lo >= hi) return;
    }
    const int64_t n0 = (int64_t)blockIdx.x * 64, k0 = (int64_t)blockIdx.y * 64, groups = k / gs;
    for (int i = threadIdx.x; i < 512; i += 256) {  // 64 rows x 8 vectors of 8 k
        const int nr = i >> 3, v = (i & 7) * 8;
        const int64_t row = n0 + nr, c = k0 + v;
        uint16_t w[8] = {};
        if (row < n) {
            const int64_t e0 = ((int64_t)expert * n + row) * k + c;
            if constexpr (ALIGNED) {
                if (c < k) {
                    const GroupPar<MODE> g = group_par<MODE>(scale, zp, ((int64_t)expert * n + row) * groups + c / gs);
                    u32v4 o;
                    if constexpr (four_bit(MODE)) o = dequant8<MODE, DT>(*(const uint32_t*)(codes + e0 / 2), 0, g, lut);
                    else {
                        const u32v2 p = *(const u32v2*)(codes + e0);
                        o = dequant8<MODE, DT>(p.x, p.y, g, lut);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[2 * j] = (uint16_t)o[j], w[2 * j + 1] = (uint16_t)(o[j] >> 16);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < k) w[j] = dequant1<MODE, DT>(codes, e0 + j, group_par<MODE>(scale, zp, (e0 + j) / gs), lut);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) tile[v + j][nr] = w[j];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 512; i += 256) {  // 64 rows of k x 8 vectors of 8 n
        const int kr = i >> 3, v = (i & 7) * 8;
        if (k0 + kr >= k || n0 + v >= np) continue;
        u32v4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = *(const uint32_t*)&tile[kr][v + 2 * j];
        *(u32v4*)(out + ((int64_t)expert * k + k0 + kr) * np + n0 + v) = o;
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
// dz = dy * act'(z) (swiglu: both halves), written with row stride ldz and zeros behind n; and the sums of dz's fp32 values
// over chunks of 32 rows, which k_sum_chunks adds up in order (no atomics: the result does not depend on the schedule).
// dz is rounded to the activations' type because the product that takes it reads 16-bit operands.
constexpr int kChunkRows = 32;
template <int DT>
__global__ __launch_bounds__(256) void k_activation_grad(const uint16_t* __restrict__ dy, int64_t ldd, const uint16_t* __restrict__ z,
                                                         int64_t m, int64_t n, int act, uint16_t* __restrict__ dz, int64_t ldz,
                                                         float* __restrict__ sums) {
    const int64_t width = act == kActSwiglu ? n / 2 : n;
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r0 = (int64_t)blockIdx.y * kChunkRows, r1 = r0 + kChunkRows < m ? r0 + kChunkRows : m;
    if (c >= width) {
        const int64_t pad = n + (c - width);  // the padding's columns, by the threads behind the last column
        if (dz && pad < ldz)
            for (int64_t r = r0; r < r1; ++r) dz[r * ldz + pad] = 0;
        return;
    }
    float s0 = 0.0f, s1 = 0.0f;
    for (int64_t r = r0; r < r1; ++r) {
        const float g = to_f32<DT>(dy[r * ldd + c]);
        float a = g;
        if (act == kActSwiglu) {
            const float zg = to_f32<DT>(z[r * n + c]), zu = to_f32<DT>(z[r * n + width + c]);
            a = g * zu * activate_grad(kActSilu, zg);
            const float b = g * zg * sigmoid_f(zg);
            s1 += b;
            if (dz) dz[r * ldz + width + c] = from_f32<DT>(b);
        } else if (act != kActNone) {
            a = g * activate_grad(act, to_f32<DT>(z[r * n + c]));
        }
        s0 += a;
        if (dz) dz[r * ldz + c] = from_f32<DT>(a);
    }
    if (sums) {
        sums[blockIdx.y * n + c] = s0;
        if (act == kActSwiglu) sums[blockIdx.y * n + width + c] = s1;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_sum_chunks(const float* __restrict__ sums, int64_t chunks, int64_t n, uint16_t* __restrict__ out) {
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= n) return;
    float s = 0.0f;
    for (int64_t i = 0; i < chunks; ++i) s += sums[i * n + c];
    out[c] = from_f32<DT>(s);
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
    const int64_t kp = round64(w.k), total_rows = w.experts * w.n, groups = w.k / w.gs;
    const bool fast = aligned_groups(w);
    const int64_t blocks = fast ? (total_rows + kDequantRows - 1) / kDequantRows : (total_rows * kp + 255) / 256;
    if (blocks > 0x7fffffff) {
        set_error("linear: weight too large");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    const uint32_t vecs = (uint32_t)(kp / 8), per_group = (uint32_t)(w.gs / 8 ? w.gs / 8 : 1);
    // ceil(2^32 / d); d == 1 would need 2^32 itself: one row of one vector, or groups of 8, take the other kernel
    const bool magic = fast && vecs > 1 && per_group > 1;
    const int64_t blocks_any = (total_rows * kp + 255) / 256;
    if (!magic && blocks_any > 0x7fffffff) {
        set_error("linear: weight too large");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    const uint32_t mr = magic ? (uint32_t)((((uint64_t)1 << 32) + vecs - 1) / vecs) : 0;
    const uint32_t mg = magic ? (uint32_t)((((uint64_t)1 << 32) + per_group - 1) / per_group) : 0;
#define GO(M)                                                                                                                  \
    if (magic)                                                                                                                 \
        hipLaunchKernelGGL((k_dequant_rows<M, DT>), dim3((unsigned)blocks), dim3(256), 0, s, w.codes, w.scale, w.zp, out, total_rows, \
                           w.n, (uint32_t)w.k, (uint32_t)kp, (uint32_t)groups, mr, mg, rows);                                 \
    else                                                                                                                       \
        hipLaunchKernelGGL((k_dequant_rows_any<M, DT>), dim3((unsigned)blocks_any), dim3(256), 0, s, w.codes, w.scale, w.zp, out, \
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
    const int64_t np = round64(w.n), tn = (w.n + 63) / 64, tk = (w.k + 63) / 64;
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
// runs on the codes themselves.
struct Need {
    size_t weight, pack;  // (the codes' product: the sums of blocks that share k in the weight's place)
    bool few;
    FewShape shape;
    size_t total() const { return weight + pack; }
};
// The time of the other way, in the units of FewShape: the weight decompressed (2.6 bytes an element at 5 TB/s) and multiplied
// by 128 x 128 or 256 x 256 tiles (1.1 and 1.7 us for 64 k of a round of blocks, the former 0.65 where half the blocks fill it).
// 28672 x 8192: codes 144 us against 280 for 128 rows, 270 against 300 for 256, 520 against 365 for 512.
int64_t dense_cost(const Weight& w, int64_t rows, bool grouped) {
    auto blocks = [&](int64_t tile) { return ((w.n + tile - 1) / tile) * ((rows + tile - 1) / tile + (grouped ? (w.experts - 1) / 2 : 0)); };
    const int64_t small = blocks(128), large = blocks(256), steps = (w.k + 63) / 64;
    const double t128 = small <= 256 ? 0.65 : 1.1 * (double)((small + 511) / 512), t256 = 1.7 * (double)((large + 255) / 256);
    const double us = (double)w.experts * (double)w.n * (double)w.k * 2.6 / 5.0e6 + (double)steps * (t128 < t256 ? t128 : t256) + 8.0;
    return (int64_t)(us / 0.12);
}
bool must_pack(const void* x, int64_t ldx, int64_t k, int64_t sources, bool gathered) {
    return k % 64 || ldx % 8 || ((uintptr_t)x & 15) || !dense_reaches(1, 32, ldx, sources, false, gathered);
}
Need forward_need(const Weight& w, const void* x, int64_t ldx, int64_t sources, bool gathered, int64_t rows, bool gated, bool grouped) {
    Need d{(size_t)(w.experts * w.n * round64(w.k)) * 2, 0, false, {}};
    const bool copy = ldx % 8 || ((uintptr_t)x & 15);
    d.few = rows <= 1024 * w.experts && few_fits(w.mode, w.k, w.gs, w.codes, copy ? rows : sources, copy ? round64(w.k) : ldx);
    if (d.few) {
        d.shape = few_plan(w.mode, w.n, w.k, w.k / w.gs, gated, rows, w.experts, grouped);
        d.few = d.shape.cost < dense_cost(w, rows, grouped);
    }
    if (d.few) {
        d.weight = d.shape.kz > 1 ? (size_t)(d.shape.kz * rows * w.n + 3) / 4 * 16 : 0;
    }
    if (d.few ? copy : must_pack(x, ldx, w.k, sources, gathered)) d.pack = (size_t)(rows * round64(w.k)) * 2;
    return d;
}
Need backward_need(const Weight& w, const void* dz, int64_t ldz, int64_t rows) {
    Need d{(size_t)(w.experts * w.k * round64(w.n)) * 2, 0, false, {}};
    if (must_pack(dz, ldz, w.n, rows, false)) d.pack = (size_t)(rows * round64(w.n)) * 2;
    return d;
}

int vec_of(const Epilogue& e) {
    const int64_t width = e.act == kActSwiglu ? e.n / 2 : e.n;
    uintptr_t bits = (uintptr_t)e.y | (uintptr_t)e.z | (uintptr_t)e.residual;
    if (e.y32 && ((uintptr_t)e.y & 15)) return 0;
    return (bits & 7) == 0 && e.ldy % 4 == 0 && (!e.residual || e.ldr % 4 == 0) && (!e.z || width % 4 == 0);
}

int pack_rows(const void*& x, int64_t& ldx, int64_t k, RowMap& rows, uint16_t* pack, hipStream_t s) {
    const int64_t kp = round64(k);
    if (rows.rows > 0x7fffffff) {
        set_error("linear: too many rows");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    hipLaunchKernelGGL(k_pack_rows, dim3((unsigned)rows.rows), dim3(256), 0, s, (const uint16_t*)x, ldx, k, kp, pack, rows);
    x = pack, ldx = kp, rows.slots = nullptr, rows.sources = rows.rows;
    return launch_status("linear: rows");
}

int run_dense(int dtype, const void* x, int64_t ldx, int64_t k, const void* w, RowMap rows, Epilogue ep, uint16_t* pack, hipStream_t s) {
    const int64_t kp = round64(k);
    if (must_pack(x, ldx, k, rows.sources, rows.slots != nullptr)) {
        const int st = pack_rows(x, ldx, k, rows, pack, s);
        if (st != NNCF_AMD_OK) return st;
    }
    if (!dense_reaches(ep.n, kp, ldx, rows.sources, ep.act == kActSwiglu, rows.slots != nullptr)) {
        set_error("linear: operands beyond the kernels' range (n=%lld k=%lld)", (long long)ep.n, (long long)k);
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
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
                                          const void* residual, int64_t ldr, void* y, int64_t ldy, void* z, void* workspace,
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
    ep.bias = bias, ep.residual = residual, ep.y = y, ep.z = z, ep.ldr = ldr, ep.ldy = ldy, ep.n = n, ep.act = activation;
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
                                      int64_t ldy, void* z, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace wc;
    const Weight w{(const uint8_t*)codes, scale, zero_point, mode, n, k, group_size == -1 ? k : group_size, experts};
    int st = check_weight("expert_linear", dtype, w);
    if (st == NNCF_AMD_OK) st = check_groups("expert_linear", offsets, slots, topk, rows, sources);
    if (st != NNCF_AMD_OK) return st;
    const RowMap map{offsets, slots, (int32_t)experts, (int32_t)topk, rows, sources};
    Epilogue ep{};
    ep.y = y, ep.z = z, ep.ldy = ldy, ep.n = n, ep.act = activation;
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

extern "C" int nncf_amd_activation_grad(const void* dy, int dtype, int64_t ldd, const void* z, int64_t m, int64_t n, int activation, void* dz,
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
    const int64_t blocks = (width + (dz ? ldz - n : 0) + 255) / 256;
    if (m > 0 && (!dy || ldd < width || (activation != kActNone && !z) || (dz && ldz < n))) {
        set_error("activation_grad: null or overlapping rows (ldd=%lld ldz=%lld)", (long long)ldd, (long long)ldz);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (chunks > 65535 || blocks > 0x7fffffff) {
        set_error("activation_grad: too many rows");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    if (dbias && m > 0 && (!workspace || workspace_bytes < nncf_amd_activation_grad_workspace(m, n))) {
        set_error("activation_grad: workspace of %zu bytes needed", nncf_amd_activation_grad_workspace(m, n));
        return NNCF_AMD_ERR_WORKSPACE;
    }
    hipStream_t s = (hipStream_t)stream;
    float* sums = dbias ? (float*)workspace : nullptr;
    if (m > 0 && (dz || dbias)) {
        const dim3 grid((unsigned)blocks, (unsigned)chunks);
        if (dtype == NNCF_AMD_BF16)
            hipLaunchKernelGGL((k_activation_grad<NNCF_AMD_BF16>), grid, dim3(256), 0, s, (const uint16_t*)dy, ldd, (const uint16_t*)z, m, n,
                               activation, (uint16_t*)dz, ldz, sums);
        else
            hipLaunchKernelGGL((k_activation_grad<NNCF_AMD_F16>), grid, dim3(256), 0, s, (const uint16_t*)dy, ldd, (const uint16_t*)z, m, n,
                               activation, (uint16_t*)dz, ldz, sums);
        const int st = launch_status("activation_grad");
        if (st != NNCF_AMD_OK) return st;
    }
    if (dbias) {
        const dim3 grid((unsigned)((n + 255) / 256));
        if (dtype == NNCF_AMD_BF16)
            hipLaunchKernelGGL((k_sum_chunks<NNCF_AMD_BF16>), grid, dim3(256), 0, s, sums, chunks, n, (uint16_t*)dbias);
        else
            hipLaunchKernelGGL((k_sum_chunks<NNCF_AMD_F16>), grid, dim3(256), 0, s, sums, chunks, n, (uint16_t*)dbias);
        return launch_status("activation_grad");
    }
    return NNCF_AMD_OK;
}
