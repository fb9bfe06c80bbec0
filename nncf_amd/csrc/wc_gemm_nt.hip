// wc_gemm_nt.hip -- y = act(x W^T + bias) + residual with W [n, k] and x [m, k] dense in the activations' 16-bit type, both
// with k running along their rows; plain or grouped by expert.  Used where the rows of x are many enough that W is worth
// decompressing once (wc_linear.hip), in both directions (the gradient takes W transposed).
//
// A block owns a tile of 64 * FA rows of W by 64 * FB rows of x, four waves in a 2 x 2 arrangement, each FA x FB
// accumulators of v_mfma_f32_32x32x16 (W is the A operand: a lane ends with four consecutive columns of one row of y).
// Both operands go global -> LDS by buffer DMA in stages of 32 k (64 bytes a row), four stages: one being read, three on
// their way.  A row's 16-byte chunk c sits at chunk position c ^ ((row >> 1) & 3): eight consecutive lanes of a fragment read
// eight rows and then touch all 32 banks once.  The DMA writes LDS linearly, so the permutation is applied to its source.
#include <type_traits>

#include "wc_linear.h"

namespace wc {

constexpr int kStages = 4;
constexpr int kRowBytes = 64;  // 32 k of 16 bits

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

// Tiles of rows: expert e has ceil(rows / PB) of them, in order.  Tile `t` -> its expert and first row; false behind the last.
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

template <int DT, int FA, int FB>
__global__ __launch_bounds__(256) void k_gemm_nt(DenseArgs g, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int PA = 64 * FA, PB = 64 * FB;  // tile rows of W and of x
    constexpr int kStageBytes = (PA + PB) * kRowBytes;
    constexpr int NDMA = FA + FB;  // DMA instructions per wave and stage: 16 rows each
    extern __shared__ __align__(16) char smem[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wi = wave >> 1, wj = wave & 1;

    // Tiles in bands of 8 row tiles, the row tile fastest inside a band; the workgroups of one XCD (they are dealt out in
    // turn over the 8 of them) take a run of consecutive tiles, so that its L2 holds 8 strips of x and a few of W.
    const uint32_t total = tiles_m * tiles_n;
    const uint32_t per = (total + 7) / 8;
    const uint32_t id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= total) return;
    const uint32_t band = id / (8 * tiles_n), in_band = id - band * 8 * tiles_n;
    const uint32_t wide = tiles_m - 8 * band < 8 ? tiles_m - 8 * band : 8;
    const uint32_t tm = 8 * band + in_band % wide, tn = in_band / wide;

    const bool gated = g.ep.act == kActSwiglu;
    const int64_t width = gated ? g.ep.n / 2 : g.ep.n;
    const int64_t col0 = (int64_t)tn * (gated ? PA / 2 : PA);

    if (g.rows.offsets) {  // rows behind the last group are zero: every row tile's block takes its share
        int64_t lo, hi;
        expert_range(g.rows, g.rows.experts - 1, lo, hi);
        const int64_t end = col0 + (gated ? PA / 2 : PA) < width ? col0 + (gated ? PA / 2 : PA) : width;
        for (int64_t r = hi + tm; r < g.rows.rows; r += tiles_m)
            for (int64_t c = col0 + threadIdx.x; c < end; c += 256) {
                if (g.ep.y32) ((float*)g.ep.y)[r * g.ep.ldy + c] = 0.0f;
                else ((uint16_t*)g.ep.y)[r * g.ep.ldy + c] = 0;
                if (g.ep.z) {
                    ((uint16_t*)g.ep.z)[r * g.ep.n + c] = 0;
                    if (gated) ((uint16_t*)g.ep.z)[r * g.ep.n + width + c] = 0;
                }
            }
    }
    int expert;
    int64_t first, last;
    if (!find_tile<PB>(g.rows, tm, expert, first, last)) return;

    // sources of this lane's DMA chunks: instruction u of the wave fills 16 consecutive tile rows
    const char* wbase = (const char*)g.w + (int64_t)expert * g.ep.n * g.k * 2;
    const char* xbase = (const char*)g.x;
    int64_t worg = 0, xorg = 0;  // origins that keep the 32-bit offsets small
    if (!gated) worg = col0;
    if (!g.rows.slots) xorg = first;
    const i32x4 rw = uniform(buffer_of(wbase + worg * g.k * 2)), rx = uniform(buffer_of(xbase + xorg * g.ldx * 2));
    uint32_t voff[NDMA], dst[NDMA];
#pragma unroll
    for (int u = 0; u < NDMA; ++u) {
        const bool is_w = u < FA;
        const uint32_t row = (is_w ? u * 64 : (u - FA) * 64) + wave * 16 + (lane >> 2);  // row in the operand's tile
        const uint32_t chunk = (lane & 3) ^ ((row >> 1) & 3);
        int64_t at;
        if (is_w) {
            int64_t c;
            if (gated) {  // a wave's rows: its gate columns, then the same columns of the other half
                const uint32_t half = 16 * FA, l = row % (32 * FA);
                c = col0 + (int64_t)(row / (32 * FA)) * half + l % half;
                c = c < width ? c : width - 1;
                if (l >= half) c += width;
            } else {
                c = col0 + row;
                c = c < width ? c : width - 1;
            }
            at = (c - worg) * g.k * 2;
        } else {
            int64_t r = first + row;
            r = r < last ? r : last - 1;
            at = (source_row(g.rows, r) - xorg) * g.ldx * 2;
        }
        voff[u] = (uint32_t)at + chunk * 16;
        dst[u] = (is_w ? 0 : PA * kRowBytes) + ((is_w ? u * 64 : (u - FA) * 64) + wave * 16) * kRowBytes;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int nst = (int)(g.k / 32);
    uint32_t so = 0, lds_st = 0;
    auto issue_prepare = [&](int st) {
        so = (uint32_t)st * kRowBytes;
        lds_st = lds0 + (uint32_t)(st % kStages) * kStageBytes;
    };
    auto issue_one = [&](int u) { dma16(u < FA ? rw : rx, voff[u], so, lds_st + dst[u]); };

    typedef int op_t __attribute__((ext_vector_type(4)));
    const uint32_t r32 = lane & 31, kh = lane >> 5;
    uint32_t offa[2], offb[2];  // per half of the stage; the fragments follow 32 rows apart (32 rows keep the permutation)
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
        const uint32_t at = r32 * kRowBytes + (((2 * ks + kh) ^ ((r32 >> 1) & 3)) * 16);
        offa[ks] = wi * 32 * FA * kRowBytes + at;
        offb[ks] = (PA + wj * 32 * FB) * kRowBytes + at;
    }
    auto read_op = [&](const char* img, uint32_t off) { return *(const op_t*)(img + off); };
    f32x16 acc[FA][FB];
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
    auto mfma = [&](f32x16& c, const op_t& a, const op_t& b) {
        if constexpr (DT == NNCF_AMD_BF16)
            asm volatile("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b) : "memory");
        else
            asm volatile("v_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b) : "memory");
    };
    auto wait_dma = [&](int stages) {  // until at most `stages` stages are on their way
        if (stages >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NDMA) : "memory");
        else if (stages == 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NDMA) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };
    constexpr int NM = FA * FB;
    constexpr int kBarrierAfter = FA + FB - 1 < NM - 1 ? FA + FB - 1 : NM - 1;
    constexpr int kSlots = 2 * NM - (kBarrierAfter + 1);
    constexpr int kSlotStep = kSlots / NDMA > 0 ? kSlots / NDMA : 1;
    static_assert(kSlots >= NDMA, "a stage's DMA instructions go between the MFMAs behind the barrier");
    op_t a0[FA], b0[FB], a1[FA], b1[FB];
    // 16 k: the MFMAs on (ca, cb); between them the LDS reads of the next 16 k, in the first half of a stage the wait for the
    // next stage and the barrier that also frees the buffer of the stage before, and behind it the DMA into that buffer
    auto kstep = [&](const op_t* ca, const op_t* cb, op_t* na, op_t* nb, const char* img, auto ks, auto reads, auto sync, auto dma,
                     int stages) {
        constexpr bool READS = decltype(reads)::value, SYNC = decltype(sync)::value, DMA = decltype(dma)::value;
        constexpr int KS = decltype(ks)::value;       // half of the stage that is read: 1 in the stage's first step, else 0
        constexpr int SLOT0 = KS == 1 ? -(kBarrierAfter + 1) : NM - (kBarrierAfter + 1);
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            mfma(acc[i / FB][i % FB], ca[i / FB], cb[i % FB]);
            if constexpr (READS) {
                if (i < FA) na[i] = read_op(img, offa[KS] + i * 32 * kRowBytes);
                else if (i < FA + FB) nb[i - FA] = read_op(img, offb[KS] + (i - FA) * 32 * kRowBytes);
                if (i == NM - 1)  // few MFMAs: the rest of the reads
#pragma unroll
                    for (int j = NM; j < FA + FB; ++j) {
                        if (j < FA) na[j] = read_op(img, offa[KS] + j * 32 * kRowBytes);
                        else nb[j - FA] = read_op(img, offb[KS] + (j - FA) * 32 * kRowBytes);
                    }
            }
            if constexpr (SYNC) {
                if (i == kBarrierAfter) {
                    wait_dma(stages);
                    __builtin_amdgcn_s_barrier();
                }
            }
            if constexpr (DMA) {
                const int slot = SLOT0 + i;
                if (slot >= 0 && slot % kSlotStep == 0 && slot / kSlotStep < NDMA) issue_one(slot / kSlotStep);
            }
        }
    };
    using T = std::true_type;
    using F = std::false_type;
    using K0 = std::integral_constant<int, 0>;
    using K1 = std::integral_constant<int, 1>;
    for (int st = 0; st < kStages - 1 && st < nst; ++st) {
        issue_prepare(st);
#pragma unroll
        for (int u = 0; u < NDMA; ++u) issue_one(u);
    }
    wait_dma((nst < kStages - 1 ? nst : kStages - 1) - 1);
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int m = 0; m < FA; ++m) a0[m] = read_op(smem, offa[0] + m * 32 * kRowBytes);
#pragma unroll
    for (int m = 0; m < FB; ++m) b0[m] = read_op(smem, offb[0] + m * 32 * kRowBytes);
    int st = 0;
    for (; st + kStages - 1 < nst; ++st) {
        const char* img = smem + (st % kStages) * kStageBytes;
        issue_prepare(st + kStages - 1);
        kstep(a0, b0, a1, b1, img, K1{}, T{}, T{}, T{}, 1);
        kstep(a1, b1, a0, b0, smem + ((st + 1) % kStages) * kStageBytes, K0{}, T{}, F{}, T{}, 0);
    }
    for (; st + 1 < nst; ++st) {
        const char* img = smem + (st % kStages) * kStageBytes;
        kstep(a0, b0, a1, b1, img, K1{}, T{}, T{}, F{}, nst - 2 - st);
        kstep(a1, b1, a0, b0, smem + ((st + 1) % kStages) * kStageBytes, K0{}, T{}, F{}, F{}, 0);
    }
    kstep(a0, b0, a1, b1, smem + (st % kStages) * kStageBytes, K1{}, T{}, F{}, F{}, 0);
    kstep(a1, b1, a0, b0, smem, K0{}, F{}, F{}, F{}, 0);
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");  // the last MFMAs leave the pipe before the read-out

    const int64_t row0 = first + wj * 32 * FB + r32;
#pragma unroll
    for (int b = 0; b < FB; ++b) {
        const int64_t row = row0 + b * 32;
        if (row >= last) continue;
        if (gated) {
#pragma unroll
            for (int a = 0; a < (FA + 1) / 2; ++a)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    __builtin_amdgcn_sched_barrier(0);
                    float s[4], u[4];
                    if constexpr (FA >= 2) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[i] = acc[a][b][4 * q + i], u[i] = acc[(a + FA / 2) % FA][b][4 * q + i];
                    }
                    finish4<DT>(g.ep, row, col0 + wi * 16 * FA + a * 32 + 8 * q + 4 * kh, s, u);
                }
        } else {
#pragma unroll
            for (int a = 0; a < FA; ++a)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    __builtin_amdgcn_sched_barrier(0);
                    float s[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[i] = acc[a][b][4 * q + i];
                    finish4<DT>(g.ep, row, col0 + wi * 32 * FA + a * 32 + 8 * q + 4 * kh, s, s);
                }
        }
    }
}

template <int DT, int FA, int FB>
int dense_tiles(const DenseArgs& a, hipStream_t s) {
    static OncePerDevice once;
    constexpr int kLds = kStages * 64 * (FA + FB) * kRowBytes;
    const int first = once.first_on_device();
    if (first < 0) {
        set_error("linear: no current device");
        return NNCF_AMD_ERR_LAUNCH;
    }
    if (first && hipFuncSetAttribute((const void*)k_gemm_nt<DT, FA, FB>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds) != hipSuccess) {
        once.forget_current();
        set_error("linear: %d bytes of LDS refused", kLds);
        return NNCF_AMD_ERR_LAUNCH;
    }
    const bool gated = a.ep.act == kActSwiglu;
    const int64_t width = gated ? a.ep.n / 2 : a.ep.n, per = gated ? 32 * FA : 64 * FA, pb = 64 * FB;
    const int64_t tiles_n = (width + per - 1) / per;
    // ragged groups: each may end inside a tile
    const int64_t groups = a.rows.offsets ? (a.rows.experts < a.rows.rows ? a.rows.experts : a.rows.rows) : 1;
    const int64_t tiles_m = a.rows.offsets ? a.rows.rows / pb + groups : (a.rows.rows + pb - 1) / pb;
    const int64_t blocks = (tiles_n * tiles_m + 7) / 8 * 8;
    if (blocks > 0x7fffffff) {
        set_error("linear: too many tiles");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    hipLaunchKernelGGL((k_gemm_nt<DT, FA, FB>), dim3((unsigned)blocks), dim3(256), kLds, s, a, (uint32_t)tiles_m, (uint32_t)tiles_n);
    return launch_status("linear");
}

bool dense_reaches(int64_t n, int64_t k, int64_t ldx, int64_t sources, bool gated, bool gathered) {
    constexpr int64_t kMost = (int64_t)0xffff0000;
    return (gated ? n : 512) * k * 2 < kMost && (gathered ? sources : 512) * ldx * 2 < kMost;
}

int dense_launch(int dtype, const DenseArgs& a, hipStream_t s) {
    if (dtype == NNCF_AMD_BF16) return dense_tiles<NNCF_AMD_BF16, 2, 2>(a, s);
    return dense_tiles<NNCF_AMD_F16, 2, 2>(a, s);
}

}  // namespace wc
