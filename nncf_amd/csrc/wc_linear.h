// wc_linear.h -- shared by the kernels that multiply activations by compressed weights (wc_linear.hip, wc_linear_few.hip,
// wc_gemm_nt.hip, wc_gemm_codes.hip, wc_experts.hip).
//
// The operator:  y[m, :] = act(x[m, :] . W^T + bias) + residual[m, :],  W [n, k] given as codes, scales and zero points.
// W is the VALUE OF THE DECOMPRESSOR in the activations' type (wc_decompress.hip), bit for bit:
//     integer modes, NF4:  RN_T(RN_fp16(d * s)),  d = code - zero point (or the code book's value in fp16), s fp16
//     MXFP4:               RN_T(e2m1 * 2^(byte - 127))
// so that a layer answers with the same weight whether it is decompressed first or multiplied as it is stored.  The sums,
// the bias, the activation and the residual are fp32; the only rounding after the products is that of y.
#pragma once
#include "wc_common.h"

namespace wc {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32v2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32v4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

enum { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActSwiglu = 5 };

// ------------------------------------------------------------------------------------------ codes -> the weight's values
// NF4's code book in fp16, as the decompressor holds it: one entry per code BYTE, the pair of its two nibbles
constexpr int kNf4Pairs = 256;
__device__ __constant__ const float kNf4Values[16] = {-1.0f, -0.6961928009986877f, -0.5250730514526367f, -0.39491748809814453f,
                                                      -0.28444138169288635f, -0.18477343022823334f, -0.09105003625154495f, 0.0f,
                                                      0.07958029955625534f, 0.16093020141124725f, 0.24611230194568634f,
                                                      0.33791524171829224f, 0.44070982933044434f, 0.5626170039176941f,
                                                      0.7229568362236023f, 1.0f};

constexpr __host__ __device__ bool four_bit(int mode) { return mode >= NNCF_AMD_INT4_ASYM; }

// what a group's scale and zero point become once: s2 the scale twice, z the zero points under the exponents that the codes
// are given (see dequant8), e8 MXFP4's power of two
template <int MODE>
struct GroupPar {
    h2 s2, z0, z1;
    float e8;
};

// from a group's raw scale (fp16 bits or E8M0 byte) and zero point
template <int MODE>
__device__ __forceinline__ GroupPar<MODE> par_of(uint32_t scale, uint32_t zero) {
    GroupPar<MODE> p{};
    if constexpr (MODE == NNCF_AMD_MXFP4) {
        p.e8 = __builtin_bit_cast(float, scale ? scale << 23 : 0x00400000u);  // byte 0: the subnormal 2^-127
    } else {
        const _Float16 s = __builtin_bit_cast(_Float16, (uint16_t)scale);
        p.s2 = h2{s, s};
        if constexpr (MODE == NNCF_AMD_INT4_SYM) zero = 8;    // codes are stored with a +8 bias
        if constexpr (MODE == NNCF_AMD_INT8_SYM) zero = 128;  // dequant8 flips the sign bit: code + 128
        if constexpr (MODE != NNCF_AMD_NF4) p.z0 = __builtin_bit_cast(h2, (0x6400u | zero) * 0x00010001u);
        if constexpr (MODE == NNCF_AMD_INT4_SYM || MODE == NNCF_AMD_INT4_ASYM)
            p.z1 = __builtin_bit_cast(h2, (0x5400u | (zero << 4)) * 0x00010001u);
    }
    return p;
}
template <int MODE>
__device__ __forceinline__ GroupPar<MODE> group_par(const void* __restrict__ scale, const uint8_t* __restrict__ zp, int64_t g) {
    uint32_t z = 0;
    if constexpr (MODE == NNCF_AMD_INT4_ASYM) z = (zp[g >> 1] >> (4 * (g & 1))) & 15u;
    if constexpr (MODE == NNCF_AMD_INT8_ASYM) z = zp[g];
    if constexpr (MODE == NNCF_AMD_MXFP4) return par_of<MODE>(((const uint8_t*)scale)[g], z);
    else return par_of<MODE>(((const uint16_t*)scale)[g], z);
}

// two fp16 values -> two of the activations' type.  fp16 -> bf16 goes through fp32 (exact) and one rounding to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pair_of(_Float16 a, _Float16 b) {
    if constexpr (DT == NNCF_AMD_F16) return __builtin_bit_cast(uint32_t, h2{a, b});
    else return __builtin_bit_cast(uint32_t, b2{(__bf16)(float)a, (__bf16)(float)b});
}
template <int DT>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
    if constexpr (DT == NNCF_AMD_F16) return __builtin_bit_cast(uint32_t, h2{(_Float16)a, (_Float16)b});
    else return __builtin_bit_cast(uint32_t, b2{(__bf16)a, (__bf16)b});
}

// 8 consecutive weights of one group: p0 (4-bit modes: 8 nibbles, the lower first) or p0, p1 (8 bytes) -> four pairs.
// (The way of codes into fp16 numbers under a fixed exponent is that of Kim et al., "Who Says Elephants Can't Run", 2022.)
// A code enters as the fp16 number 1024 + c (its bits under the exponent 0x6400) or, where it sits four bits higher, as
// 64 + c under 0x5400 (the units there are sixteenths), which saves the shift; the difference to 1024 + z or 64 + z is
// exact and the packed product rounds once, as the decompressor does.
template <int MODE, int DT>
__device__ __forceinline__ u32v4 dequant8(uint32_t p0, uint32_t p1, const GroupPar<MODE>& g, const h2* lut) {
    u32v4 r;
    if constexpr (MODE == NNCF_AMD_MXFP4) {
        if constexpr (DT == NNCF_AMD_BF16) {
            r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, g.e8, 0));
            r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, g.e8, 1));
            r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, g.e8, 2));
            r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(p0, g.e8, 3));
        } else {
            r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(p0, g.e8, 0));
            r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(p0, g.e8, 1));
            r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(p0, g.e8, 2));
            r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(p0, g.e8, 3));
        }
    } else if constexpr (MODE == NNCF_AMD_NF4) {
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const h2 v = lut[(p0 >> (8 * k)) & 255u] * g.s2;
            o[k] = pair_of<DT>(v.x, v.y);
        }
        r = u32v4{o[0], o[1], o[2], o[3]};
    } else if constexpr (MODE == NNCF_AMD_INT4_SYM || MODE == NNCF_AMD_INT4_ASYM) {
        // masks in scalar and exponents in vector registers: one v_and_or_b32 each (as literals they take two instructions)
        uint32_t m0 = 0x000f000fu, m1 = 0x00f000f0u, e0 = 0x64006400u, e1 = 0x54005400u;
        asm("" : "+s"(m0), "+s"(m1), "+v"(e0), "+v"(e1));
        const uint32_t q = p0 >> 8;
        const h2 a = (__builtin_bit_cast(h2, (p0 & m0) | e0) - g.z0) * g.s2;  // elements 0, 4
        const h2 b = (__builtin_bit_cast(h2, (p0 & m1) | e1) - g.z1) * g.s2;  // 1, 5
        const h2 c = (__builtin_bit_cast(h2, (q & m0) | e0) - g.z0) * g.s2;   // 2, 6
        const h2 d = (__builtin_bit_cast(h2, (q & m1) | e1) - g.z1) * g.s2;   // 3, 7
        r = u32v4{pair_of<DT>(a.x, b.x), pair_of<DT>(c.x, d.x), pair_of<DT>(a.y, b.y), pair_of<DT>(c.y, d.y)};
    } else {
        uint32_t w[2] = {p0, p1};
        if constexpr (MODE == NNCF_AMD_INT8_SYM) {
            w[0] ^= 0x80808080u;
            w[1] ^= 0x80808080u;
        }
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t sel = (k & 1) ? 0x03070106u : 0x03050104u;  // bytes under the exponent byte 0x64
            const h2 v = (__builtin_bit_cast(h2, __builtin_amdgcn_perm(w[k >> 1], 0x64006400u, sel)) - g.z0) * g.s2;
            o[k] = pair_of<DT>(v.x, v.y);
        }
        r = u32v4{o[0], o[1], o[2], o[3]};
    }
    return r;
}

// one weight by its place (odd shapes)
template <int MODE, int DT>
__device__ __forceinline__ uint16_t dequant1(const uint8_t* __restrict__ codes, int64_t e, const GroupPar<MODE>& g, const h2* lut) {
    uint32_t c;
    if constexpr (four_bit(MODE)) c = (codes[e >> 1] >> (4 * (e & 1))) & 15u;
    else c = codes[e];
    return (uint16_t)dequant8<MODE, DT>(c, 0, g, lut).x;
}

template <int MODE>
__device__ __forceinline__ void fill_nf4(h2* lut) {
    if constexpr (MODE == NNCF_AMD_NF4) {
        for (int i = threadIdx.x; i < kNf4Pairs; i += blockDim.x)
            lut[i] = h2{(_Float16)kNf4Values[i & 15], (_Float16)kNf4Values[i >> 4]};
        __syncthreads();
    }
}

// ----------------------------------------------------------------------------------------------------------- activations
// sigmoid as 1 / (1 + e^-z): e^-z = inf for z < -88 gives 0, the limit
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }
constexpr float kGeluC = 1.5957691216057308f;  // 2 * sqrt(2 / pi): tanh(u) written as 2 * sigmoid(2 u) - 1

// Phi(z), the normal distribution's integral.  Its left tail is e^(-z^2 / 2) t P(t) with t = 1 / (1 + 0.46 |z| / sqrt(2)) in (0, 1],
// P the polynomial of degree 7 that is closest, in relative terms, to e^(z^2 / 2) Phi(-|z|) / t over the whole of that interval
// (least squares with weights raised where the error is largest, until it is level: 6.8e-7).  So the tail is off by a share of
// ITSELF -- 1e-6 up to |z| = 4, 9e-6 at 13, where the rounding of z^2 / 2 is what counts -- and gelu's only rounding that shows
// in 16 bits is that of y.  (A fit of the absolute error, Abramowitz and Stegun 7.1.26, is 0.05 % off at -4 and 1 % at -8 for
// two products less; the library's erfcf takes about 100 instructions, 20 us of the epilogue of 2047 x 4096 results.)
__device__ __forceinline__ float normal_cdf(float z) {
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(fabsf(z), 0.32526913f, 1.0f));
    float p = 0.033857215f;
    p = __builtin_fmaf(p, t, -0.113314785f);
    p = __builtin_fmaf(p, t, 0.08459569f);
    p = __builtin_fmaf(p, t, 0.026305184f);
    p = __builtin_fmaf(p, t, 0.09342394f);
    p = __builtin_fmaf(p, t, 0.11559094f);
    p = __builtin_fmaf(p, t, 0.12977864f);
    p = __builtin_fmaf(p, t, 0.12976353f);
    const float tail = p * t * __expf(-0.5f * z * z);
    return z > 0.0f ? 1.0f - tail : tail;
}

__device__ __forceinline__ float activate(int act, float z) {
    switch (act) {
        case kActRelu: return z > 0.0f ? z : (z == z ? 0.0f : z);
        case kActGelu: return z * normal_cdf(z);
        case kActGeluTanh: return z * sigmoid_f(kGeluC * (z + 0.044715f * z * z * z));
        case kActSilu: return z * sigmoid_f(z);
        default: return z;
    }
}
__device__ __forceinline__ float activate_grad(int act, float z) {
    // far out every derivative has reached its limit; there z * z would overflow and meet a zero (a NaN passes)
    z = z > 1e4f ? 1e4f : (z < -1e4f ? -1e4f : z);
    switch (act) {
        case kActRelu: return z > 0.0f ? 1.0f : 0.0f;
        case kActGelu: return normal_cdf(z) + z * __expf(-0.5f * z * z) * 0.3989422804014327f;
        case kActGeluTanh: {
            const float s = sigmoid_f(kGeluC * (z + 0.044715f * z * z * z));
            return s + z * s * (1.0f - s) * kGeluC * (1.0f + 0.134145f * z * z);
        }
        case kActSilu: {
            const float s = sigmoid_f(z);
            return s + z * s * (1.0f - s);
        }
        default: return 1.0f;
    }
}

template <int DT>
__device__ __forceinline__ float to_f32(uint16_t v) {
    if constexpr (DT == NNCF_AMD_F16) return (float)__builtin_bit_cast(_Float16, v);
    else return __builtin_bit_cast(float, (uint32_t)v << 16);
}
template <int DT>
__device__ __forceinline__ uint16_t from_f32(float v) {
    if constexpr (DT == NNCF_AMD_F16) return __builtin_bit_cast(uint16_t, (_Float16)v);
    else return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// --------------------------------------------------------------------------------------------------------------- problem
// Where rows come from and how they are grouped.  offsets == nullptr: one weight, `rows` rows.  Else expert e owns the rows
// [offsets[e], offsets[e + 1]) and the rows behind offsets[experts] get zeros.  slots != nullptr: row r reads x at
// slots[r] / topk.  Both arrays are read with their values held to what the buffers have, so that a handle with other numbers
// in it cannot reach memory that is not its own.
struct RowMap {
    const int32_t* offsets;
    const int32_t* slots;
    int32_t experts, topk;
    int64_t rows, sources;  // rows of y; rows of x
};
__device__ __forceinline__ int64_t held(int64_t v, int64_t lo, int64_t hi) { return v < lo ? lo : (v > hi ? hi : v); }
__device__ __forceinline__ void expert_range(const RowMap& r, int e, int64_t& lo, int64_t& hi) {
    if (!r.offsets) {
        lo = 0, hi = r.rows;
        return;
    }
    lo = held(r.offsets[e], 0, r.rows);
    hi = held(r.offsets[e + 1], lo, r.rows);
}
__device__ __forceinline__ int64_t source_row(const RowMap& r, int64_t row) {
    if (!r.slots) return row;
    const int32_t s = r.slots[row];
    return held((int64_t)((uint32_t)(s < 0 ? 0 : s) / (uint32_t)r.topk), 0, r.sources - 1);
}

struct Epilogue {
    const void* bias;      // [n] or null
    const void* residual;  // [rows, width] or null
    void* y;               // [rows, width]
    float* slope;          // [rows, n] or null: what the gradient of a row's sums takes dy times (`slopes`)
    int64_t ldr, ldy, n;   // n: rows of the weight; swiglu: gate rows first, width = n / 2
    int act;
    int y32;               // y is fp32 (gradients that are summed over rows afterwards)
    int vec;               // 4 consecutive columns may be stored at once (y, residual, slope and their row strides allow it)
};

// The activation's derivative in place of the sum z (swiglu: those of both halves, z and u, in their places).  They are kept in
// fp32: in 16 bits, they or the sums, they double the rounding error of the bias' gradient (bf16: 0.0031 for 0.0017 of its norm).
__device__ __forceinline__ void slopes(int act, float& z, float& u) {
    const float at = z;
    if (act == kActSwiglu) z = u * activate_grad(kActSilu, at), u = at * sigmoid_f(at);
    else z = activate_grad(act, at);
}

// up to four consecutive columns of one row; `up` only for swiglu (a: the gate's sums, b: the other half's)
template <int DT>
__device__ __forceinline__ void finish4(const Epilogue& e, int64_t row, int64_t col, const float* a, const float* b) {
    const int64_t width = e.act == kActSwiglu ? e.n / 2 : e.n;
    if (col >= width) return;
    const int cnt = width - col < 4 ? (int)(width - col) : 4;
    float z[4], u[4], v[4];
    const uint16_t* bias = (const uint16_t*)e.bias;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        z[i] = a[i];
        u[i] = e.act == kActSwiglu ? b[i] : 0.0f;
        if (bias && i < cnt) {
            z[i] += to_f32<DT>(bias[col + i]);
            if (e.act == kActSwiglu) u[i] += to_f32<DT>(bias[width + col + i]);
        }
        __builtin_amdgcn_sched_barrier(0);  // one after the other: side by side their exponentials need the most registers
        v[i] = e.act == kActSwiglu ? z[i] * sigmoid_f(z[i]) * u[i] : activate(e.act, z[i]);
        if (e.slope) slopes(e.act, z[i], u[i]);
    }
    uint16_t* y = (uint16_t*)e.y + row * e.ldy + col;
    const uint16_t* res = e.residual ? (const uint16_t*)e.residual + row * e.ldr + col : nullptr;
    float* so = e.slope ? e.slope + row * e.n + col : nullptr;
    if (e.y32) {
        float* y32 = (float*)e.y + row * e.ldy + col;
        if (e.vec && cnt == 4) *(f32x4*)y32 = f32x4{v[0], v[1], v[2], v[3]};
        else
            for (int i = 0; i < cnt; ++i) y32[i] = v[i];
        return;
    }
    if (e.vec && cnt == 4) {
        if (res) {
            const u32v2 r = *(const u32v2*)res;
            v[0] += to_f32<DT>((uint16_t)r.x), v[1] += to_f32<DT>((uint16_t)(r.x >> 16));
            v[2] += to_f32<DT>((uint16_t)r.y), v[3] += to_f32<DT>((uint16_t)(r.y >> 16));
        }
        *(u32v2*)y = u32v2{pair_of<DT>(v[0], v[1]), pair_of<DT>(v[2], v[3])};
        if (so) {
            *(f32x4*)so = f32x4{z[0], z[1], z[2], z[3]};
            if (e.act == kActSwiglu) *(f32x4*)(so + width) = f32x4{u[0], u[1], u[2], u[3]};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= cnt) break;
        if (res) v[i] += to_f32<DT>(res[i]);
        y[i] = from_f32<DT>(v[i]);
        if (so) {
            so[i] = z[i];
            if (e.act == kActSwiglu) so[width + i] = u[i];
        }
    }
}

// the product of dense operands (wc_gemm_nt.hip): x [sources, ldx] with k a multiple of 64, 192 at least, and 16-byte rows,
// w [experts * n, k]
struct DenseArgs {
    const void* x;
    const void* w;
    int64_t ldx, k;
    RowMap rows;
    Epilogue ep;
};
// true where the tile kernels can address the operands (32-bit offsets from a tile's origin)
bool dense_reaches(int64_t n, int64_t k, int64_t ldx, int64_t sources, bool gated, bool gathered);
int dense_launch(int dtype, const DenseArgs& a, hipStream_t s);

// the product for few rows per group, from the codes (wc_linear_few.hip): rows of whole 32 k, groups of 32, of whole 64 or the
// row, 16-byte rows of x
struct FewArgs {
    const void* x;
    int64_t ldx;
    const uint8_t* codes;
    const void* scale;
    const uint8_t* zp;
    uint32_t k, groups, magic;  // groups per row; magic: ceil(2^32 / (group size / 16))
    uint32_t scales8;           // ceil(2^32 / (groups / 8)) where rows have whole eight groups, aligned in memory; else 0
    RowMap rows;
    Epilogue ep;
    float* sums;                // [kz][rows][n], kz > 1
};
// A block's shape and its LDS: codes [wave][2 KiB] (at the end the waves' sums), x [buffer][part][row][512 bytes (8-bit codes:
// 256)], scales [strip][group][16 rows], zero points.
struct FewShape {
    int wn, wk, rows, buffers;    // rows of x at a time
    int lds_rows, tiles;          // and that LDS holds; tiles of 16 of them
    int steps, per_wk;            // steps of a wave; ceil(2^16 / wk)
    int kz;                       // blocks that share k: above 1 they leave fp32 sums [kz][rows][n] in the workspace
    int pitch;                    // groups of a row, and a place behind them (groups of 32: two, a quarter reads both)
    int scale_bytes, zero_bytes;  // per group; zero_bytes 0: none
    int x_bytes;                  // of a row and step
    int64_t cost;                 // its time in units of 0.12 us
    __host__ __device__ int waves() const { return wn * wk; }
    __host__ __device__ int x() const { return waves() * 2048; }
    __host__ __device__ int scales() const {  // the waves' sums take the place of codes and x
        const int end = x() + buffers * wk * lds_rows * x_bytes, sums = waves() * tiles * 1024;
        return end > sums ? end : sums;
    }
    __host__ __device__ int zeros() const { return scales() + (wn * 16 * pitch * scale_bytes + 15) / 16 * 16; }
    __host__ __device__ int total() const { return zeros() + wn * 16 * pitch * zero_bytes; }
};

bool few_fits(int mode, int64_t k, int64_t gs, const void* codes, int64_t sources, int64_t ldx);
// the quickest shape for `rows` rows of x over `experts` weights (grouped: with row offsets)
FewShape few_plan(int mode, int64_t n, int64_t k, int64_t groups, bool gated, int64_t rows, int64_t experts, bool grouped);
int few_launch(int dtype, int mode, const FewArgs& a, const FewShape& sh, hipStream_t s);
int lds_refused(int bytes);  // the error of a launcher whose opt-in to so much LDS failed
// y from the sums [kz][rows][n] that blocks sharing k left, in the order of their parts
int join_sums(int dtype, const float* sums, int kz, const RowMap& rows, const Epilogue& ep, hipStream_t s);

// the product by tiles, from the codes (wc_gemm_codes.hip): k a multiple of 64, groups of 32, of whole 64 or the row, x as for
// the dense product
struct CodesArgs {
    const void* x;
    int64_t ldx, k;
    const uint8_t* codes;
    const void* scale;
    const uint8_t* zp;
    uint32_t groups, group_stages;  // per row; stages of 64 k per group (0: groups of 32)
    uint64_t magic;                 // ceil(2^32 / group_stages)
    RowMap rows;
    Epilogue ep;
    float* sums;  // [kz][rows][n], kz > 1
    int kz;
};
struct CodesShape {
    int fb, kz;  // tiles of 128 fb rows of x; blocks that share k
    double us;
};
bool codes_fits(int mode, int64_t n, int64_t k, int64_t gs, const void* codes);
CodesShape codes_plan(int mode, int64_t n, int64_t k, bool gated, int64_t rows, int64_t experts, bool grouped);
int codes_launch(int dtype, int mode, int fb, const CodesArgs& a, hipStream_t s);

}  // namespace wc
