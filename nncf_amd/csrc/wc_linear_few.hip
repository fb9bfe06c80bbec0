// wc_linear_few.hip -- the product with a compressed weight for few rows of x (a token per sequence): up to 16 of them, or as many
// per expert, at a time.  Bound by the bytes of the codes (0.5-1 per weight), which are read once and dequantised in registers.
//
// A block owns 16 * R rows of W; its waves take consecutive parts of k and add their sums through LDS.  A lane holds row
// (lane & 15) and 32 consecutive k of a step of 128 (the four quarters of the wave side by side): one 16-byte load of 4-bit
// codes, all of one group.  That is the A operand of four v_mfma_f32_16x16x32 whose B operand is the same 32 k of x's row
// (lane & 15): the order of k inside a step is free as long as both operands share it.  The codes, scales and x of the next
// step are requested before the current one is used.
#include "wc_linear.h"

namespace wc {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kFewWaves = 8;

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32v4& a, const u32v4& b, f32x4 c) {
    if constexpr (DT == NNCF_AMD_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int MODE, int R>
struct FewStep {
    u32v4 codes[R][four_bit(MODE) ? 1 : 2];
    uint32_t scale[R], zero[R];
    u32v4 x[4];
};

template <int MODE, int DT, int R>
__global__ __launch_bounds__(64 * kFewWaves, 4) void k_few_rows(FewArgs a) {
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    __shared__ f32x4 part[kFewWaves][R][64];
    fill_nf4<MODE>(lut);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int r16 = lane & 15, kq = lane >> 4;
    const int expert = blockIdx.y;
    const bool gated = a.ep.act == kActSwiglu;
    const int64_t n = a.ep.n, width = gated ? n / 2 : n;
    const int tiles = gated ? R / 2 : R;  // tiles of 16 columns of y
    const int64_t col0 = (int64_t)blockIdx.x * 16 * tiles;
    int64_t lo, hi;
    if (a.rows.offsets && expert == 0) {  // rows behind the last group are zero
        expert_range(a.rows, a.rows.experts - 1, lo, hi);
        for (int64_t r = hi + wave; r < a.rows.rows; r += kFewWaves)
            if (lane < 16 * tiles && col0 + lane < width) {
                ((uint16_t*)a.ep.y)[r * a.ep.ldy + col0 + lane] = 0;
                if (a.ep.z) {
                    ((uint16_t*)a.ep.z)[r * n + col0 + lane] = 0;
                    if (gated) ((uint16_t*)a.ep.z)[r * n + width + col0 + lane] = 0;
                }
            }
    }
    expert_range(a.rows, expert, lo, hi);
    if (lo >= hi) return;

    const uint32_t k = a.k, steps = (k + 127) / 128, per_wave = (steps + kFewWaves - 1) / kFewWaves;
    const uint32_t s0 = wave * per_wave, s1 = s0 + per_wave < steps ? s0 + per_wave : steps;
    const uint8_t* code_at[R];
    int64_t group_at[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        int64_t c = col0 + (gated ? r % (R > 1 ? R / 2 : 1) : r) * 16 + r16;
        c = c < width ? c : width - 1;
        if (gated && r >= R / 2) c += width;
        const int64_t row = (int64_t)expert * n + c;
        code_at[r] = a.codes + (four_bit(MODE) ? row * k / 2 : row * k);
        group_at[r] = row * a.groups;
    }
    for (int64_t t0 = lo; t0 < hi; t0 += 16) {
        const bool live = t0 + r16 < hi;
        const uint16_t* xrow = (const uint16_t*)a.x + (live ? source_row(a.rows, t0 + r16) : 0) * a.ldx;
        f32x4 acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = f32x4{0, 0, 0, 0};

        FewStep<MODE, R> st[2];
        auto load = [&](uint32_t s, FewStep<MODE, R>& d) {
            uint32_t at = s * 128 + kq * 32;
            const bool in = at < k;  // the last step may be short: its lanes read place 0 and count as zero through x
            at = in ? at : 0;
            const uint32_t v = at / 32, g = a.magic ? __umulhi(v, a.magic) : v;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if constexpr (four_bit(MODE)) {
                    d.codes[r][0] = *(const u32v4*)(code_at[r] + at / 2);
                } else {
                    d.codes[r][0] = *(const u32v4*)(code_at[r] + at);
                    d.codes[r][1] = *(const u32v4*)(code_at[r] + at + 16);
                }
                const int64_t gi = group_at[r] + g;
                if constexpr (MODE == NNCF_AMD_MXFP4) d.scale[r] = ((const uint8_t*)a.scale)[gi];
                else d.scale[r] = ((const uint16_t*)a.scale)[gi];
                d.scale[r] = in ? d.scale[r] : 0;
                if constexpr (MODE == NNCF_AMD_INT4_ASYM) d.zero[r] = (uint32_t)(a.zp[gi >> 1] >> (4 * (gi & 1))) & 15u;
                if constexpr (MODE == NNCF_AMD_INT8_ASYM) d.zero[r] = a.zp[gi];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) d.x[j] = u32v4{0, 0, 0, 0};
            if (live && in) {
#pragma unroll
                for (int j = 0; j < 4; ++j) d.x[j] = *(const u32v4*)(xrow + at + 8 * j);
            }
        };
        auto use = [&](const FewStep<MODE, R>& d) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const GroupPar<MODE> g = par_of<MODE>(d.scale[r], d.zero[r]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    u32v4 w;
                    if constexpr (four_bit(MODE)) w = dequant8<MODE, DT>(d.codes[r][0][j], 0, g, lut);
                    else w = dequant8<MODE, DT>(d.codes[r][j >> 1][2 * (j & 1)], d.codes[r][j >> 1][2 * (j & 1) + 1], g, lut);
                    acc[r] = mfma16<DT>(w, d.x[j], acc[r]);
                }
            }
        };
        if (s0 < s1) {
            load(s0, st[0]);
            uint32_t s = s0;
            for (; s + 2 < s1; s += 2) {
                load(s + 1, st[1]);
                use(st[0]);
                load(s + 2, st[0]);
                use(st[1]);
            }
            if (s + 1 < s1) {
                load(s + 1, st[1]);
                use(st[0]);
                use(st[1]);
            } else {
                use(st[0]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) part[wave][r][lane] = acc[r];
        __syncthreads();
        if (wave < tiles) {
            f32x4 s = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kFewWaves; ++w) {
                s += part[w][wave][lane];
                if (gated) u += part[w][(wave + R / 2) % R][lane];
            }
            if (t0 + r16 < hi) {
                const float sv[4] = {s.x, s.y, s.z, s.w}, uv[4] = {u.x, u.y, u.z, u.w};
                finish4<DT>(a.ep, t0 + r16, col0 + wave * 16 + 4 * kq, sv, uv);
            }
        }
        __syncthreads();
    }
}

bool few_fits(int mode, int64_t k, int64_t gs, const void* codes) {
    return k % 32 == 0 && gs % 32 == 0 && k <= (1 << 20) && ((uintptr_t)codes & 15) == 0 && mode <= NNCF_AMD_MXFP4;
}

template <int DT>
int few_typed(int mode, const FewArgs& a, hipStream_t s) {
    const bool gated = a.ep.act == kActSwiglu;
    const int64_t width = gated ? a.ep.n / 2 : a.ep.n;
    const int64_t tiles = (width + 15) / 16;
    // two tiles of rows per wave read x half as often; one where that would leave compute units without a block
    const int r = gated || tiles * a.rows.experts >= 1024 ? 2 : 1;
    const int64_t per = gated ? r / 2 : r;
    const int64_t gx = (tiles + per - 1) / per;
    if (gx > 0x7fffffff || a.rows.experts > 65535) {
        set_error("linear: weight too large");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    const dim3 grid((unsigned)gx, (unsigned)a.rows.experts), block(64 * kFewWaves);
#define GO(M)                                                                                  \
    case M:                                                                                    \
        if (r == 2) hipLaunchKernelGGL((k_few_rows<M, DT, 2>), grid, block, 0, s, a);          \
        else hipLaunchKernelGGL((k_few_rows<M, DT, 1>), grid, block, 0, s, a);                 \
        break;
    switch (mode) {
        GO(NNCF_AMD_INT8_ASYM)
        GO(NNCF_AMD_INT8_SYM)
        GO(NNCF_AMD_INT4_ASYM)
        GO(NNCF_AMD_INT4_SYM)
        GO(NNCF_AMD_NF4)
        GO(NNCF_AMD_MXFP4)
    }
#undef GO
    return launch_status("linear");
}

int few_launch(int dtype, int mode, const FewArgs& a, hipStream_t s) {
    return dtype == NNCF_AMD_BF16 ? few_typed<NNCF_AMD_BF16>(mode, a, s) : few_typed<NNCF_AMD_F16>(mode, a, s);
}

}  // namespace wc
