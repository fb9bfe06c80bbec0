// wc_linear_few.hip -- the product with a compressed weight for few rows of x (a token per sequence, a small batch): up to 64 of
// them, or as many per expert, at a time.  The codes (0.5-1 byte per weight) are read once and dequantised in registers.
//
// A block owns WN strips of 16 rows of W and cuts k into WK parts, one wave for each pair (up to 16), all in step; one block per
// compute unit where the strips allow it, so that there is one start and one end.  A wave's step is 256 k (128 with 8-bit
// codes) of its strip: 16 rows x 128 bytes, whole lines, eight lanes a row (a load straight into the operand's layout, 16 rows
// x 64 bytes, reaches 3.3 TB/s on a 28672 x 8192 weight, this one 5.0), turned round in 2 KiB of LDS of the wave's own; the
// rows' 16-byte chunks are permuted (c ^ (row >> 1)) so that both sides touch all banks.  From there a lane takes 8 bytes of row
// (lane & 15) at a time: the A operand of one (8-bit codes) or two v_mfma_f32_16x16x32.  The codes of the next two steps are
// on their way meanwhile.
// x, four to eight times the codes' bytes if every strip read it by itself and in the operand's scattered order, comes to LDS in
// whole rows, once for the waves that share a part of k, a step ahead (two buffers, one barrier a step).  The strips' scales
// and zero points, one run of memory, come to LDS at the start: a scattered load of two bytes a lane takes the load unit about
// as many cycles as it has lanes.
//
// One token over 4096 x 4096 int4 takes 7.8 us (1.1 TB/s of codes: start and end), over 28672 x 8192 44 us (2.7 TB/s), 16 tokens
// with asymmetric codes and the gate 52: bound there by the vector instructions of the conversion (13.7 clocks a weight and
// lane, 20 us) and what a step adds to them.  Five tokens that hit five of eight mxfp4 experts of 28672 x 4096 (one instruction a
// pair) 85 us, 3.4 TB/s of the codes that are hit; seven of them 108 us, 3.8.
#include <type_traits>

#include "wc_linear.h"

namespace wc {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kFewWaves = 16;
constexpr int kFewLdsBytes = 160 * 1024 - 1024;  // less the NF4 table

template <int DT>
__device__ __forceinline__ f32x4 mfma16(const u32v4& a, const u32v4& b, f32x4 c) {
    if constexpr (DT == NNCF_AMD_BF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// TT: tiles of 16 rows of x.  XI: loads of two rows of x (8-bit codes: four) that a wave makes per step; 8 of them need the
// registers of 16 waves for 8.
template <int MODE, int DT, int TT, int XI>
__global__ __launch_bounds__(XI == 8 ? 512 : 1024, XI == 8 ? 2 : 4) void k_few_rows(FewArgs a, FewShape sh) {
    constexpr int MF = four_bit(MODE) ? 2 : 1;           // matrix instructions per 8 bytes of codes
    constexpr uint32_t KS = four_bit(MODE) ? 256 : 128;  // k of a step
    constexpr int XROWS = 1024 / (2 * KS);               // rows of x per load, 16 bytes a lane
    constexpr bool ASYM = MODE == NNCF_AMD_INT4_ASYM || MODE == NNCF_AMD_INT8_ASYM;
    using scale_t = typename std::conditional<MODE == NNCF_AMD_MXFP4, uint8_t, uint16_t>::type;
    __shared__ h2 lut[MODE == NNCF_AMD_NF4 ? kNf4Pairs : 1];
    extern __shared__ __align__(16) char dyn[];
    fill_nf4<MODE>(lut);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wn = wave * sh.per_wk >> 16, wk = wave - wn * sh.wk;
    char* mine = dyn + wave * 2048;
    char* xbuf = dyn + sh.x();
    scale_t* scales = (scale_t*)(dyn + sh.scales());
    uint8_t* zeros = (uint8_t*)(dyn + sh.zeros());
    const int expert = blockIdx.y;
    const bool gated = a.ep.act == kActSwiglu;
    const int64_t n = a.ep.n, width = gated ? n / 2 : n;
    // strip w of the block: 16 columns of y; with a gate the even ones are the gate's rows, the odd ones the other half's
    auto column_of = [&](int w) { return gated ? ((int64_t)blockIdx.x * (sh.wn / 2) + (w >> 1)) * 16 : ((int64_t)blockIdx.x * sh.wn + w) * 16; };
    int64_t lo, hi;
    if (a.rows.offsets && expert == 0 && blockIdx.z == 0) {  // rows behind the last group are zero
        expert_range(a.rows, a.rows.experts - 1, lo, hi);
        const int64_t c0 = column_of(0), c1 = c0 + (gated ? sh.wn / 2 : sh.wn) * 16 < width ? c0 + (gated ? sh.wn / 2 : sh.wn) * 16 : width;
        for (int64_t r = hi + wave; r < a.rows.rows; r += sh.waves())
            for (int64_t c = c0 + lane; c < c1; c += 64) {
                ((uint16_t*)a.ep.y)[r * a.ep.ldy + c] = 0;
                if (a.ep.slope) {
                    a.ep.slope[r * n + c] = 0.0f;
                    if (gated) a.ep.slope[r * n + width + c] = 0.0f;
                }
            }
    }
    expert_range(a.rows, expert, lo, hi);
    if (lo >= hi) return;

    const uint32_t k = a.k, steps = sh.steps;
    const uint32_t row_bytes = four_bit(MODE) ? k / 2 : k;
    // Blocks begin at different places of k and go round: all in step at one column, they would ask the few memory channels
    // that hold it (rows are often a power of two apart).
    const uint32_t turn = (blockIdx.x & 15) * steps >> 4;
    auto stage_of = [&](uint32_t s) {
        uint32_t t = s + turn;
        t = t < steps ? t : t - steps;
        return (blockIdx.z * steps + (t < steps ? t : 0)) * sh.wk + wk;
    };
    // rows of W from a scalar origin; rows behind the last are held to it, strips behind the last read the last row
    auto origin_of = [&](int w) {
        const int64_t c = column_of(w);
        return (int64_t)expert * n + (c < width ? c : width - 1) + (gated && (w & 1) ? width : 0);
    };
    auto held_row = [&](int w, int i) {
        const int64_t left = width - 1 - column_of(w);
        return (uint32_t)(left < 0 ? 0 : i < left ? i : left);
    };
    const uint8_t* codes0 = a.codes + origin_of(wn) * row_bytes;
    bool fresh = true;  // the scales are not yet here
    for (int64_t t0 = lo; t0 < hi; t0 += sh.rows) {
        const int rows = (int)(hi - t0 < sh.rows ? hi - t0 : sh.rows);
        // (the lane's number anew: what is computed from it must not be carried round this loop in registers)
        int lane = threadIdx.x & 63;
        asm volatile("" : "+v"(lane));
        const int r16 = lane & 15, kq = lane >> 4;
        const uint32_t lc = (lane & 7) * 16;
        const uint32_t ra = held_row(wn, lane >> 3) * row_bytes, rb = held_row(wn, (lane >> 3) + 8) * row_bytes;
        const int put = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 4)) << 4);  // rows lane / 8 and 8 further: (row >> 1) & 7
        const int put8 = ((lane >> 3) + 8) * 128 + (((lane & 7) ^ ((lane >> 4) + 4)) << 4);
        const int get = r16 * 128 + (kq & 1) * 8;
        u32v4 codes[2][2];
        auto load = [&](uint32_t s, int d) {  // step s of this wave: the parts of k take turns
            uint32_t at = stage_of(s) * 128 + lc;
            at = at < row_bytes ? at : 0;  // behind the end: the row's first codes, times x's zeros
            codes[d][0] = __builtin_nontemporal_load((const u32v4*)(codes0 + (ra + at)));
            codes[d][1] = __builtin_nontemporal_load((const u32v4*)(codes0 + (rb + at)));
        };
        load(0, 0);
        load(1, 1);
        // this wave's loads of x: rows wn * XROWS + lane / (64 / XROWS), then WN * XROWS further; those behind the last are held to it
        uint32_t x_src[XI];
        int x_put[XI];
        const int xc = lane & (64 / XROWS - 1);
#pragma unroll
        for (int i = 0; i < XI; ++i) {
            int r = (wn + i * sh.wn) * XROWS + lane / (64 / XROWS);
            r = r < rows ? r : rows - 1;
            x_src[i] = (uint32_t)(source_row(a.rows, t0 + r) * a.ldx);
            x_put[i] = (wk * sh.lds_rows + r) * sh.x_bytes + ((xc ^ (r & 7)) << 4);
        }
        u32v4 xr[XI];
        auto load_x = [&](uint32_t s) {
            uint32_t at = stage_of(s) * KS + xc * 8;
            at = at < k ? at : 0;
#pragma unroll
            for (int i = 0; i < XI; ++i) xr[i] = *(const u32v4*)((const uint16_t*)a.x + (x_src[i] + at));
        };
        const int x_size = sh.buffers > 1 ? sh.wk * sh.lds_rows * sh.x_bytes : 0;
        auto put_x = [&](uint32_t s) {
            if (stage_of(s) * KS + KS > k) {  // what lies behind the end of k counts as zero
                const bool in = stage_of(s) * KS + xc * 8 < k;
#pragma unroll
                for (int i = 0; i < XI; ++i) xr[i] = in ? xr[i] : u32v4{0, 0, 0, 0};
            }
#pragma unroll
            for (int i = 0; i < XI; ++i) *(u32v4*)(xbuf + (s & 1) * x_size + x_put[i]) = xr[i];
        };
        load_x(0);
        if (fresh) {
            // many loads at a time: a loop over single ones would wait for each
            auto put_scale = [&](int at, uint32_t v) { scales[at] = (scale_t)v; };
            if (a.scales8) {  // rows of whole eight groups: 8 of them a thread
                const uint32_t eights = a.groups / 8, all = sh.wn * 16 * eights;
                for (uint32_t i0 = threadIdx.x; i0 < all; i0 += 2 * blockDim.x) {
                    u32v4 v[2];
                    uint32_t at[2];
                    u32v2 zv[2];
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const uint32_t i = i0 + u * blockDim.x < all ? i0 + u * blockDim.x : i0, r = __umulhi(i, a.scales8), e = i - r * eights;
                        const int64_t g0 = (origin_of(r >> 4) + held_row(r >> 4, r & 15)) * a.groups + e * 8;
                        if constexpr (sizeof(scale_t) == 1) {
                            const u32v2 w = *(const u32v2*)((const uint8_t*)a.scale + g0);
                            v[u] = u32v4{w.x, w.y, 0, 0};
                        } else {
                            v[u] = *(const u32v4*)((const uint16_t*)a.scale + g0);
                        }
                        if constexpr (MODE == NNCF_AMD_INT4_ASYM) zv[u].x = *(const uint32_t*)(a.zp + (g0 >> 1));
                        if constexpr (MODE == NNCF_AMD_INT8_ASYM) zv[u] = *(const u32v2*)(a.zp + g0);
                        at[u] = ((r >> 4) * sh.pitch + e * 8) * 16 + (r & 15);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const uint32_t w = sizeof(scale_t) == 1 ? v[u][j >> 2] >> (8 * (j & 3)) : v[u][j >> 1] >> (16 * (j & 1));
                            put_scale(at[u] + j * 16, w);
                            if constexpr (MODE == NNCF_AMD_INT4_ASYM) zeros[at[u] + j * 16] = (zv[u].x >> (4 * j)) & 15;
                            if constexpr (MODE == NNCF_AMD_INT8_ASYM) zeros[at[u] + j * 16] = (uint8_t)(zv[u][j >> 2] >> (8 * (j & 3)));
                        }
                }
            } else {
                for (uint32_t g0 = 0; g0 < a.groups; g0 += 4) {  // a thread per row: lanes follow the rows of W
                    for (int r = threadIdx.x; r < sh.wn * 16; r += blockDim.x) {
                        const int64_t row = (origin_of(r >> 4) + held_row(r >> 4, r & 15)) * a.groups;
                        uint32_t v[4], z[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int64_t g = row + (g0 + j < a.groups ? g0 + j : a.groups - 1);
                            v[j] = ((const scale_t*)a.scale)[g];
                            if constexpr (MODE == NNCF_AMD_INT4_ASYM) z[j] = (a.zp[g >> 1] >> (4 * (g & 1))) & 15;
                            if constexpr (MODE == NNCF_AMD_INT8_ASYM) z[j] = a.zp[g];
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (g0 + j < a.groups) {
                                put_scale(((r >> 4) * sh.pitch + g0 + j) * 16 + (r & 15), v[j]);
                                if constexpr (ASYM) zeros[((r >> 4) * sh.pitch + g0 + j) * 16 + (r & 15)] = (uint8_t)z[j];
                            }
                    }
                }
            }
            // What lies behind the last group, half a quarter of an odd number of groups of 32 among it, has scale 0: whatever
            // codes stand there, their values are finite and meet x's zeros (under another group's scale they could be infinite).
            for (uint32_t g = a.groups; g < (uint32_t)sh.pitch; ++g)
                for (int r = threadIdx.x; r < sh.wn * 16; r += blockDim.x) {
                    put_scale(((r >> 4) * sh.pitch + g) * 16 + (r & 15), 0);
                    if constexpr (ASYM) zeros[((r >> 4) * sh.pitch + g) * 16 + (r & 15)] = 0;
                }
        }
        fresh = false;
        put_x(0);
        load_x(1);
        auto sync = [&] {  // LDS only: the loads stay on their way
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        sync();
        // rows behind the last: their columns are not stored (what LDS holds there reaches nothing else)
        const int xrow = TT > 1 || r16 < rows ? r16 : rows - 1;
        // x's 16-byte chunk of a quarter: its low three bits are permuted by the row; whole 128 bytes are added on top
        uint32_t x_get[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            x_get[h] = (wk * sh.lds_rows + xrow) * sh.x_bytes + (((MF == 2 ? kq * 2 + h : kq + 4 * h) ^ (xrow & 7)) << 4);
        // a quarter lies in one group, the same for all lanes but with groups of 32 (4-bit codes), where it takes in two
        const int group0 = (wn * sh.pitch + (MF == 2 && a.groups * 32 == k ? kq >> 1 : 0)) * 16 + r16;
        f32x4 acc[TT];
#pragma unroll
        for (int j = 0; j < TT; ++j) acc[j] = f32x4{0, 0, 0, 0};
        constexpr int kTile = 16 * (four_bit(MODE) ? 512 : 256);  // bytes of 16 rows of x
        auto step = [&](uint32_t s, int d) {
            *(u32v4*)(mine + put) = codes[d][0];
            *(u32v4*)(mine + put8) = codes[d][1];
            load(s + 2, d);
            const char* xs = xbuf + (s & 1) * x_size;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t kk = stage_of(s) * KS + q * (KS / 4), at = __umulhi(kk / 16, a.magic);
                const int gi = group0 + 16 * (int)(at < a.groups ? at : a.groups);  // (behind the end of k: scale 0)
                const GroupPar<MODE> g = par_of<MODE>(scales[gi], ASYM ? zeros[gi] : 0);
                const u32v2 c = *(const u32v2*)(mine + get + (((2 * q + (kq >> 1)) ^ (r16 >> 1)) << 4));
                if constexpr (MF == 2) {
                    const u32v4 w0 = dequant8<MODE, DT>(c.x, 0, g, lut), w1 = dequant8<MODE, DT>(c.y, 0, g, lut);
#pragma unroll
                    for (int j = 0; j < TT; ++j) {
                        acc[j] = mfma16<DT>(w0, *(const u32v4*)(xs + x_get[0] + q * 128 + j * kTile), acc[j]);
                        acc[j] = mfma16<DT>(w1, *(const u32v4*)(xs + x_get[1] + q * 128 + j * kTile), acc[j]);
                    }
                } else {
                    const u32v4 w0 = dequant8<MODE, DT>(c.x, c.y, g, lut);
#pragma unroll
                    for (int j = 0; j < TT; ++j) acc[j] = mfma16<DT>(w0, *(const u32v4*)(xs + x_get[q & 1] + (q >> 1) * 128 + j * kTile), acc[j]);
                }
                __builtin_amdgcn_sched_barrier(0);  // interleaved further, the values need more registers than there are
            }
            if (s + 1 < steps) {  // (uniform over the block)
                put_x(s + 1);
                load_x(s + 2);
            }
            sync();
        };
        uint32_t s = 0;
        for (; s + 1 < steps; s += 2) {
            step(s, 0);
            step(s + 1, 1);
        }
        if (s < steps) step(s, 0);
        f32x4* sums = (f32x4*)dyn;  // [wave][tile][lane]; every wave is behind its last step
#pragma unroll
        for (int j = 0; j < TT; ++j) sums[(wave * TT + j) * 64 + lane] = acc[j];
        sync();
        if (!(gated && (wn & 1))) {
            asm volatile("" : "+v"(lane));
            const int r16 = lane & 15, kq = lane >> 4;
            for (int j = wk; j < TT; j += sh.wk) {
                if (16 * j >= rows) break;
                f32x4 v = {0, 0, 0, 0}, u = {0, 0, 0, 0};
#pragma unroll 4
                for (int w = 0; w < sh.wk; ++w) {
                    v += sums[((wn * sh.wk + w) * TT + j) * 64 + lane];
                    if (gated) u += sums[(((wn + 1) * sh.wk + w) * TT + j) * 64 + lane];
                }
                if (16 * j + r16 < rows) {
                    const float vv[4] = {v.x, v.y, v.z, v.w}, uv[4] = {u.x, u.y, u.z, u.w};
                    const int64_t row = t0 + 16 * j + r16, col = column_of(wn) + 4 * kq;
                    if (sh.kz == 1) {
                        finish4<DT>(a.ep, row, col, vv, uv);
                    } else {
                        float* to = a.sums + ((int64_t)blockIdx.z * a.rows.rows + row) * n + col;
                        for (int i = 0; i < 4 && col + i < width; ++i) {
                            to[i] = vv[i];
                            if (gated) to[width + i] = uv[i];
                        }
                    }
                }
            }
        }
        sync();
    }
}

// the blocks' sums over the parts of k, in their order, and the epilogue: a thread per 4 columns of a row
template <int DT>
__global__ __launch_bounds__(256) void k_join_sums(const float* __restrict__ sums, int kz, RowMap rows, Epilogue ep) {
    const int64_t width = ep.act == kActSwiglu ? ep.n / 2 : ep.n;
    const int64_t quads = (width + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    int64_t lo, end = rows.rows;
    if (rows.offsets) expert_range(rows, rows.experts - 1, lo, end);
    const int64_t row = i / quads, col = (i - row * quads) * 4;
    if (row >= end) return;  // (rows behind the last group have their zeros)
    float s[4] = {0, 0, 0, 0}, u[4] = {0, 0, 0, 0};
    for (int z = 0; z < kz; ++z) {
        const float* from = sums + ((int64_t)z * rows.rows + row) * ep.n + col;
        if (col + 4 <= width && ep.n % 4 == 0 && width % 4 == 0) {
            const f32x4 v = *(const f32x4*)from;
            s[0] += v.x, s[1] += v.y, s[2] += v.z, s[3] += v.w;
            if (ep.act == kActSwiglu) {
                const f32x4 w = *(const f32x4*)(from + width);
                u[0] += w.x, u[1] += w.y, u[2] += w.z, u[3] += w.w;
            }
        } else {
            for (int j = 0; j < 4 && col + j < width; ++j) {
                s[j] += from[j];
                if (ep.act == kActSwiglu) u[j] += from[width + j];
            }
        }
    }
    finish4<DT>(ep, row, col, s, u);
}

int join_sums(int dtype, const float* sums, int kz, const RowMap& rows, const Epilogue& ep, hipStream_t s) {
    const int64_t width = ep.act == kActSwiglu ? ep.n / 2 : ep.n, blocks = ((width + 3) / 4 * rows.rows + 255) / 256;
    if (blocks > 0x7fffffff) {
        set_error("linear: too many rows");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    if (dtype == NNCF_AMD_BF16) hipLaunchKernelGGL((k_join_sums<NNCF_AMD_BF16>), dim3((unsigned)blocks), dim3(256), 0, s, sums, kz, rows, ep);
    else hipLaunchKernelGGL((k_join_sums<NNCF_AMD_F16>), dim3((unsigned)blocks), dim3(256), 0, s, sums, kz, rows, ep);
    return launch_status("linear");
}

FewShape few_shape(int mode, int64_t k, int64_t groups, int wn, int wk, int kz, int rows, int tiles) {
    const bool four = four_bit(mode);
    const int64_t stages = (k + (four ? 255 : 127)) / (four ? 256 : 128);
    const int steps = (int)((stages + (int64_t)wk * kz - 1) / ((int64_t)wk * kz));
    return FewShape{wn, wk, rows, steps > 1 ? 2 : 1, tiles > 1 ? 16 * tiles : rows, tiles, steps, (65536 + wk - 1) / wk, kz, (int)groups + (groups * 32 == k ? 2 : 1),
                    mode == NNCF_AMD_MXFP4 ? 1 : 2, mode == NNCF_AMD_INT4_ASYM || mode == NNCF_AMD_INT8_ASYM ? 1 : 0, four ? 512 : 256, 0};
}

int few_loads(int mode, const FewShape& sh) {  // of x, per wave and step
    const int per_load = four_bit(mode) ? 2 : 4;
    return (sh.rows + sh.wn * per_load - 1) / (sh.wn * per_load);
}

bool few_fits(int mode, int64_t k, int64_t gs, const void* codes, int64_t sources, int64_t ldx) {
    return k % 32 == 0 && (gs == k || gs % 64 == 0 || gs == 32) && k <= (1 << 20) && few_shape(mode, k, k / gs, 2, 1, 1, 16, 1).total() <= kFewLdsBytes && ((uintptr_t)codes & 15) == 0 && mode <= NNCF_AMD_MXFP4 &&
           sources * ldx < ((int64_t)1 << 31);
}

static FewShape search(int mode, int64_t n, int64_t k, int64_t groups, bool gated, int64_t rows, int64_t experts, bool grouped) {
    const int64_t strips = ((gated ? n / 2 : n) + 15) / 16 * (gated ? 2 : 1);
    const int64_t stage = four_bit(mode) ? 256 : 128, stages = (k + stage - 1) / stage;
    // rows per group: with experts the mean, a quarter more for their spread
    const int64_t most = grouped ? (rows < 16 ? rows : (5 * rows / experts + 3) / 4) : rows;
    FewShape best{};
    best.cost = INT64_MAX;
    for (int tiles = 1; tiles <= 4; tiles *= 2) {
        if (tiles > 1 && most <= 8 * tiles) break;
        const int64_t passes = (most + 16 * tiles - 1) / (16 * tiles);
        const int64_t held = grouped ? (rows < 16 * tiles ? rows : 16 * tiles) : (rows + passes - 1) / passes;  // passes of equal length
        for (int wn = gated ? 2 : 1; wn <= 8; wn += gated ? 2 : 1)
            for (int wk = 1; wn * wk <= kFewWaves && wk <= stages; ++wk)
                for (int kz = 1; kz <= 16 && (kz == 1 || kz * wk <= stages); kz += kz < 4 ? 1 : kz < 8 ? 2 : 4) {
                    const FewShape sh = few_shape(mode, k, groups, wn, wk, kz, (int)held, tiles);
                    const int loads = few_loads(mode, sh);
                    if (sh.total() > kFewLdsBytes || loads > 8 || (loads > 4 && wn * wk > kFewWaves / 2)) continue;
                    // In units of 0.12 us, from 28672 x 8192 and 4096 x 4096: a step takes 6 and 1 for every wave on the compute unit,
                    // a tenth more with two tiles of x and six tenths with four; a round of blocks 40 to start and end; the join
                    // of kz blocks 25 and its bytes.
                    const int waves_fit = kFewWaves / sh.waves(), lds_fit = kFewLdsBytes / sh.total();
                    const int64_t blocks = (strips + wn - 1) / wn * experts * kz;
                    int64_t per_cu = waves_fit < lds_fit ? waves_fit : lds_fit;
                    const int64_t rounds = (blocks + 256 * per_cu - 1) / (256 * per_cu);
                    if (blocks < 256 * per_cu) per_cu = (blocks + 255) / 256;
                    const int64_t step = (6 + per_cu * sh.waves()) * (tiles == 1 ? 10 : tiles == 2 ? 11 : 16);
                    int64_t cost = rounds * (passes * (sh.steps + 1) * step / 10 + 40);
                    if (kz > 1) cost += 25 + kz * rows * n / 60000;
                    if (cost < best.cost) best = sh, best.cost = cost;
                }
    }
    return best;
}

// The search takes tens of microseconds; its answers depend on these numbers alone and are kept, per thread.
FewShape few_plan(int mode, int64_t n, int64_t k, int64_t groups, bool gated, int64_t rows, int64_t experts, bool grouped) {
    struct Known {
        int64_t key[7];
        FewShape shape;
    };
    static thread_local Known known[64];
    const int64_t key[7] = {n, k, groups, rows, experts, mode * 4 + gated * 2 + grouped, 1};
    uint64_t h = 0;
    for (int64_t v : key) h = (h ^ (uint64_t)v) * 0x9e3779b97f4a7c15ull, h ^= h >> 29;
    Known& at = known[h & 63];
    for (int i = 0; i < 7; ++i)
        if (at.key[i] != key[i]) {
            at.shape = search(mode, n, k, groups, gated, rows, experts, grouped);
            for (int j = 0; j < 7; ++j) at.key[j] = key[j];
            break;
        }
    return at.shape;
}

template <int MODE, int DT, int TT, int XI>
int few_start(const FewArgs& a, const FewShape& sh, hipStream_t s) {
    static OncePerDevice once;
    const bool gated = a.ep.act == kActSwiglu;
    const int64_t width = gated ? a.ep.n / 2 : a.ep.n, strips = (width + 15) / 16 * (gated ? 2 : 1);
    const int64_t blocks = (strips + sh.wn - 1) / sh.wn;
    const bool opted_in = once.run([&] {
        return hipFuncSetAttribute((const void*)k_few_rows<MODE, DT, TT, XI>, hipFuncAttributeMaxDynamicSharedMemorySize, kFewLdsBytes) == hipSuccess;
    });
    if (!opted_in) return lds_refused(kFewLdsBytes);
    if (blocks > 0x7fffffff || a.rows.experts > 65535) {
        set_error("linear: weight too large");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    const dim3 grid((unsigned)blocks, (unsigned)a.rows.experts, (unsigned)sh.kz);
    hipLaunchKernelGGL((k_few_rows<MODE, DT, TT, XI>), grid, dim3(64 * sh.waves()), (size_t)sh.total(), s, a, sh);
    const int st = launch_status("linear");
    if (st != NNCF_AMD_OK || sh.kz == 1) return st;
    return join_sums(DT, a.sums, sh.kz, a.rows, a.ep, s);
}

template <int MODE, int DT>
int few_go(const FewArgs& a, const FewShape& sh, hipStream_t s) {
    const int loads = few_loads(MODE, sh);
    if (sh.tiles == 1) {
        if (loads <= 1) return few_start<MODE, DT, 1, 1>(a, sh, s);
        if (loads <= 4) return few_start<MODE, DT, 1, 4>(a, sh, s);
        return few_start<MODE, DT, 1, 8>(a, sh, s);
    }
    if (sh.tiles == 2) return loads <= 4 ? few_start<MODE, DT, 2, 4>(a, sh, s) : few_start<MODE, DT, 2, 8>(a, sh, s);
    return loads <= 4 ? few_start<MODE, DT, 4, 4>(a, sh, s) : few_start<MODE, DT, 4, 8>(a, sh, s);
}

template <int DT>
int few_typed(int mode, const FewArgs& a, const FewShape& sh, hipStream_t s) {
    switch (mode) {
        case NNCF_AMD_INT8_ASYM: return few_go<NNCF_AMD_INT8_ASYM, DT>(a, sh, s);
        case NNCF_AMD_INT8_SYM: return few_go<NNCF_AMD_INT8_SYM, DT>(a, sh, s);
        case NNCF_AMD_INT4_ASYM: return few_go<NNCF_AMD_INT4_ASYM, DT>(a, sh, s);
        case NNCF_AMD_INT4_SYM: return few_go<NNCF_AMD_INT4_SYM, DT>(a, sh, s);
        case NNCF_AMD_NF4: return few_go<NNCF_AMD_NF4, DT>(a, sh, s);
        default: return few_go<NNCF_AMD_MXFP4, DT>(a, sh, s);
    }
}

int few_launch(int dtype, int mode, const FewArgs& a, const FewShape& sh, hipStream_t s) {
    return dtype == NNCF_AMD_BF16 ? few_typed<NNCF_AMD_BF16>(mode, a, sh, s) : few_typed<NNCF_AMD_F16>(mode, a, sh, s);
}

}  // namespace wc
