// wc_gemm.h -- what the tile products (wc_gemm_nt.hip: dense operands, wc_gemm_codes.hip: the weight as codes) share: the DMA
// into LDS, ragged groups as tiles, and the way from the accumulators to y.
#pragma once
#include "wc_linear.h"

namespace wc {

constexpr int kRowBytes = 128;  // 64 k of 16 bits

// written out: through the builtin the compiler sees an LDS store of unknown address and waits for it at every LDS read
__device__ __forceinline__ void dma16(const i32x4& rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(rsrc), "s"(soff), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ i32x4 buffer_of(const void* base) {
    const uint64_t b = (uint64_t)base;
    return i32x4{(int)(uint32_t)b, (int)(uint32_t)(b >> 32), -1, 0x00020000};
}
__device__ __forceinline__ i32x4 uniform(i32x4 v) {
    return i32x4{__builtin_amdgcn_readfirstlane(v.x), __builtin_amdgcn_readfirstlane(v.y), __builtin_amdgcn_readfirstlane(v.z),
                 __builtin_amdgcn_readfirstlane(v.w)};
}
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// Tiles of rows: expert e has ceil(rows / PB) of them, in order.  How many there are, `most` at most.
template <int PB>
__device__ __forceinline__ uint32_t count_tiles(const RowMap& r, uint32_t most) {
    const int lane = threadIdx.x & 63;
    int64_t sum = 0;
    for (int e = lane; e < r.experts; e += 64) {
        int64_t lo, hi;
        expert_range(r, e, lo, hi);
        sum += (hi - lo + PB - 1) / PB;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) sum += __shfl_xor(sum, d, 64);
    return (uint32_t)uniform(sum < (int64_t)most ? sum : (int64_t)most);
}
// Tile `t` -> its expert and first row; false behind the last.
template <int PB>
__device__ __forceinline__ bool find_tile(const RowMap& r, int64_t t, int& expert, int64_t& first, int64_t& last) {
    if (!r.offsets) {
        expert = 0, first = t * PB, last = r.rows;
        return first < last;
    }
    const int lane = threadIdx.x & 63;
    for (int e0 = 0; e0 < r.experts; e0 += 64) {  // 64 experts at a time: prefix sum over the wave
        int64_t lo = 0, hi = 0;
        if (e0 + lane < r.experts) expert_range(r, e0 + lane, lo, hi);
        const int tiles = (int)((hi - lo + PB - 1) / PB);
        int sum = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d, 64);
            if (lane >= d) sum += v;
        }
        const int total = __shfl(sum, 63, 64);
        if (t < total) {
            const int at = __ffsll((unsigned long long)__ballot(sum > t)) - 1;
            const int before = __shfl(sum - tiles, at, 64);
            const int64_t lo_at = ((int64_t)__shfl((int)(lo >> 32), at, 64) << 32) | (uint32_t)__shfl((int)lo, at, 64);
            const int64_t hi_at = ((int64_t)__shfl((int)(hi >> 32), at, 64) << 32) | (uint32_t)__shfl((int)hi, at, 64);
            expert = __builtin_amdgcn_readfirstlane(e0 + at);
            first = lo_at + (t - before) * PB;
            last = hi_at;
            return true;
        }
        t -= total;
    }
    return false;
}

// rows behind the last group are zero: block (tn, tm) of a grid of tiles takes its columns of every tiles_m-th of them
template <int THREADS>
__device__ __forceinline__ void zero_rows(const RowMap& rows, const Epilogue& e, uint32_t tn, uint32_t tm, uint32_t tiles_m, int cols) {
    const bool gated = e.act == kActSwiglu;
    const int64_t width = gated ? e.n / 2 : e.n, col = (int64_t)tn * cols, end = col + cols < width ? col + cols : width;
    int64_t lo, hi;
    expert_range(rows, rows.experts - 1, lo, hi);
    if (tm >= tiles_m) return;
    for (int64_t r = hi + tm; r < rows.rows; r += tiles_m)
        for (int64_t c = col + threadIdx.x; c < end; c += THREADS) {
            if (e.y32) ((float*)e.y)[r * e.ldy + c] = 0.0f;
            else ((uint16_t*)e.y)[r * e.ldy + c] = 0;
            if (e.slope) {
                e.slope[r * e.n + c] = 0.0f;
                if (gated) e.slope[r * e.n + width + c] = 0.0f;
            }
        }
}

// 32 rows of sums in LDS -> y, where all the columns are inside and their addresses allow vectors: LANES lanes per row, 8
// columns each, so that a lane keeps its columns' bias, and four of its rows of the residual are requested before the first is needed.
template <int DT, int ACT, int LANES, int PITCH>
__device__ __forceinline__ void finish_rows(const Epilogue& e, const float* tile, int64_t row0, int64_t last, int64_t col0, uint32_t lane) {
    typedef uint32_t halves8 __attribute__((ext_vector_type(4), aligned(8)));
    constexpr bool GATED = ACT == kActSwiglu;
    constexpr int ROWS = 64 / LANES, TURNS = 32 / ROWS, AT_ONCE = TURNS < 4 ? TURNS : 4;
    const int64_t width = GATED ? e.n / 2 : e.n, col = col0 + lane % LANES * 8;
    const uint32_t r0 = lane / LANES;
    float bz[8] = {}, bu[GATED ? 8 : 1] = {};
    if (e.bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            bz[i] = to_f32<DT>(((const uint16_t*)e.bias)[col + i]);
            if constexpr (GATED) bu[i] = to_f32<DT>(((const uint16_t*)e.bias)[width + col + i]);
        }
    }
    auto pack = [](const float* v) { return halves8{pair_of<DT>(v[0], v[1]), pair_of<DT>(v[2], v[3]), pair_of<DT>(v[4], v[5]), pair_of<DT>(v[6], v[7])}; };
#pragma unroll 1
    for (int t0 = 0; t0 < TURNS; t0 += AT_ONCE) {
        halves8 res[AT_ONCE];
        if (e.residual) {
#pragma unroll
            for (int t = 0; t < AT_ONCE; ++t) {
                const int64_t row = row0 + (t0 + t) * ROWS + r0;
                res[t] = *(const halves8*)((const uint16_t*)e.residual + (row < last ? row : last - 1) * e.ldr + col);
            }
        }
#pragma unroll
        for (int t = 0; t < AT_ONCE; ++t) {
            const uint32_t r = (t0 + t) * ROWS + r0;
            const int64_t row = row0 + r;
            const float* at = tile + r * PITCH + lane % LANES * 8;
            float z[8], u[GATED ? 8 : 1] = {}, v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[i] = at[i] + bz[i];
                if constexpr (GATED) u[i] = at[LANES * 8 + i] + bu[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (GATED) v[i] = z[i] * sigmoid_f(z[i]) * u[i];
                else v[i] = activate(ACT, z[i]);
            }
            if (row >= last) continue;
            if (e.y32) {
                float* y = (float*)e.y + row * e.ldy + col;
                *(f32x4*)y = f32x4{v[0], v[1], v[2], v[3]}, *(f32x4*)(y + 4) = f32x4{v[4], v[5], v[6], v[7]};
                continue;
            }
            if (e.residual) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[2 * j] += to_f32<DT>((uint16_t)res[t][j]), v[2 * j + 1] += to_f32<DT>((uint16_t)(res[t][j] >> 16));
            }
            *(halves8*)((uint16_t*)e.y + row * e.ldy + col) = pack(v);
            if (e.slope) {
                float* to = e.slope + row * e.n + col;
#pragma unroll
                for (int i = 0; i < 8; ++i) slopes(ACT, z[i], u[GATED ? i : 0]);
                *(f32x4*)to = f32x4{z[0], z[1], z[2], z[3]}, *(f32x4*)(to + 4) = f32x4{z[4], z[5], z[6], z[7]};
                if constexpr (GATED)
                    *(f32x4*)(to + width) = f32x4{u[0], u[1], u[2], u[3]}, *(f32x4*)(to + width + 4) = f32x4{u[4], u[5], u[6], u[7]};
            }
        }
    }
}

// Through LDS, 32 rows of y at a time (a wave's own 32 x 32 FA floats, rows 16 bytes further apart than they are long), so
// that a row's columns are finished and stored side by side and the epilogue is in the program once per 32 rows.
template <int FA>
constexpr int kTileFloats = 32 * (32 * FA + 4);
template <int DT, int FA, int FB>
__device__ __forceinline__ void store_tile(const Epilogue& e, const f32x16 (&acc)[FA][FB], float* tile, int64_t row_w, int64_t last,
                                           int64_t col_w, uint32_t lane) {
    constexpr int kPitch = 32 * FA + 4;
    const bool gated = e.act == kActSwiglu;
    const int64_t width = gated ? e.n / 2 : e.n;
    const uint32_t cols = gated ? 16 * FA : 32 * FA, r32 = lane & 31, kh = lane >> 5;
    const bool whole = e.vec && col_w + cols <= width;
    __syncthreads();
#pragma unroll 1
    for (int b = 0; b < FB; ++b) {
#pragma unroll
        for (int bb = 0; bb < FB; ++bb) {
            if (bb != b) continue;
#pragma unroll
            for (int a = 0; a < FA; ++a)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *(f32x4*)(tile + r32 * kPitch + a * 32 + 8 * q + 4 * kh) =
                        f32x4{acc[a][bb][4 * q], acc[a][bb][4 * q + 1], acc[a][bb][4 * q + 2], acc[a][bb][4 * q + 3]};
        }
        const int64_t row0 = row_w + b * 32;  // (the wave's own floats: no barrier)
        if (row0 >= last) break;
        if (whole) {
#define FINISH(ACT, LANES) \
    case ACT: finish_rows<DT, ACT, LANES, kPitch>(e, tile, row0, last, col_w, lane); break;
            switch (e.act) {
                FINISH(kActNone, 4 * FA)
                FINISH(kActRelu, 4 * FA)
                FINISH(kActGelu, 4 * FA)
                FINISH(kActGeluTanh, 4 * FA)
                FINISH(kActSilu, 4 * FA)
                FINISH(kActSwiglu, 2 * FA)
            }
#undef FINISH
            continue;
        }
        for (uint32_t i = lane * 4; i < 32 * cols; i += 256) {
            const uint32_t r = i / cols, c = i % cols;
            if (row0 + r >= last) break;
            const f32x4 s = *(const f32x4*)(tile + r * kPitch + c);
            const f32x4 u = gated ? *(const f32x4*)(tile + r * kPitch + 16 * FA + c) : s;
            const float sv[4] = {s.x, s.y, s.z, s.w}, uv[4] = {u.x, u.y, u.z, u.w};
            finish4<DT>(e, row0 + r, col_w + c, sv, uv);
        }
    }
}

}  // namespace wc
