// wc_gemm_nt.hip -- y = act(x W^T + bias) + residual with W [n, k] and x [m, k] dense in the activations' 16-bit type, both
// with k running along their rows; plain or grouped by expert.  Used where the rows of x are many enough that W is worth
// decompressing once (wc_linear.hip), in both directions (the gradient takes W transposed).
//
// A block owns a tile of 32 * WI * FA rows of W by 32 * WJ * FB rows of x, WI x WJ waves, each FA x FB accumulators of
// v_mfma_f32_32x32x16 (W is the A operand: a lane ends with four consecutive columns of one row of y).
// Both operands go global -> LDS by buffer DMA in stages of 64 k: 128 bytes a row, whole lines (stages of 32 k ask for half
// lines and fetch each of them twice).  LDS has five slots for stages of one operand: while a stage is read, the next one and
// W's of the one after land; a barrier in the last quarter of a stage frees it (two slots per operand: 645 us against 600 for
// 2000 gathered rows over eight experts of 4096 x 14336).  A row's 16-byte chunk c sits at chunk position c ^ (row / 2 & 7): 16
// consecutive lanes of a fragment read 16 rows and touch all 64 banks.  The DMA writes LDS linearly, so the permutation is
// applied to its source.
//
// A stage of 64 k takes 2250 clocks of the 2048 that its matrix instructions need; what bounds it is power: the clock goes down
// to 1.6-1.7 GHz while it runs (2.1 with the DMA taken out).  The epilogue takes 5 us a tile, 8 columns per lane (30 us when each
// lane took 4 and chose the activation per element).
#include <type_traits>

#include "wc_gemm.h"

namespace wc {

constexpr int kSlots = 5;  // of LDS: a stage of one operand each

template <int DT, int WI, int WJ, int FA, int FB>
__global__ __launch_bounds__(64 * WI * WJ) void k_gemm_nt(DenseArgs g, uint32_t tiles_m, uint32_t tiles_n) {
    constexpr int NW = WI * WJ, PA = 32 * WI * FA, PB = 32 * WJ * FB;  // waves; tile rows of W and of x
    static_assert(PA == PB, "the operands' stages take each other's slots");
    constexpr int kSlotBytes = PA * kRowBytes;
    constexpr int DA = PA / (8 * NW), DB = PB / (8 * NW), NDMA = DA + DB;  // DMA instructions per wave and stage: 8 rows each
    static_assert(PA % (8 * NW) == 0 && PB % (8 * NW) == 0, "every wave brings in whole instructions' rows");
    extern __shared__ __align__(16) char smem[];
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wi = wave / WJ, wj = wave % WJ;

    const bool gated = g.ep.act == kActSwiglu;
    const int64_t width = gated ? g.ep.n / 2 : g.ep.n;
    if (g.rows.offsets) {  // rows behind the last group are zero: every block of the grid takes its share
        zero_rows<64 * NW>(g.rows, g.ep, blockIdx.x % tiles_n, blockIdx.x / tiles_n, tiles_m, gated ? PA / 2 : PA);
        tiles_m = count_tiles<PB>(g.rows, tiles_m);
    }

    // Tiles in bands of 8 row tiles, the row tile fastest inside a band; the workgroups of one XCD (they are dealt out in
    // turn over the 8 of them) take a run of consecutive tiles, so that its L2 holds 8 strips of x and a few of W.  Ragged
    // groups: of the tiles that there are, since the grid has as many as there could be.
    const uint32_t total = tiles_m * tiles_n;
    const uint32_t per = (total + 7) / 8;
    const uint32_t id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= total) return;
    const uint32_t band = id / (8 * tiles_n), in_band = id - band * 8 * tiles_n;
    const uint32_t wide = tiles_m - 8 * band < 8 ? tiles_m - 8 * band : 8;
    const uint32_t tm = 8 * band + in_band % wide, tn = in_band / wide;
    const int64_t col0 = (int64_t)tn * (gated ? PA / 2 : PA);

    int expert;
    int64_t first, last;
    if (!find_tile<PB>(g.rows, tm, expert, first, last)) return;
    first = uniform(first), last = uniform(last);

    // sources of this lane's DMA chunks: instruction u of the wave fills 8 consecutive tile rows
    const char* wbase = (const char*)g.w + (int64_t)expert * g.ep.n * g.k * 2;
    const char* xbase = (const char*)g.x;
    int64_t worg = 0, xorg = 0;  // origins that keep the 32-bit offsets small
    if (!gated) worg = col0;
    if (!g.rows.slots) xorg = first;
    const i32x4 rw = uniform(buffer_of(wbase + worg * g.k * 2)), rx = uniform(buffer_of(xbase + xorg * g.ldx * 2));
    uint32_t voff[NDMA], dst[NDMA];
#pragma unroll
    for (int u = 0; u < NDMA; ++u) {
        const bool is_w = u < DA;
        const uint32_t at8 = ((is_w ? u : u - DA) * NW + wave) * 8, row = at8 + (lane >> 3);  // row in the operand's tile
        const uint32_t chunk = (lane & 7) ^ (row >> 1 & 7);
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
        dst[u] = at8 * kRowBytes;
    }
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    const int nst = (int)(g.k / 64);
    // Slots of a stage, going round: W's 2 st, x's 2 st + 1 (modulo 5).  So W's stage may come in one stage earlier than x's.
    uint32_t so_w = 0, so_x = 0, slot_w = 0, slot_x = 0;
    auto issue_prepare = [&](int st_x, int st_w) {  // x's stage and W's stage that are brought in next
        so_x = (uint32_t)st_x * kRowBytes, so_w = (uint32_t)st_w * kRowBytes;
        slot_x = lds0 + (uint32_t)(2 * st_x + 1) % kSlots * kSlotBytes, slot_w = lds0 + (uint32_t)(2 * st_w) % kSlots * kSlotBytes;
    };
    // u < DB: x's instructions, then W's
    auto issue_one = [&](int u) {
        if (u < DB) dma16(rx, voff[DA + u], so_x, slot_x + dst[DA + u]);
        else dma16(rw, voff[u - DB], so_w, slot_w + dst[u - DB]);
    };

    typedef int op_t __attribute__((ext_vector_type(4)));
    const uint32_t r32 = lane & 31, kh = lane >> 5;
    uint32_t offa[4], offb[4];  // per quarter of the stage; the fragments follow 32 rows apart (32 rows keep the permutation)
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        const uint32_t at = r32 * kRowBytes + (((2 * ks + kh) ^ (r32 >> 1 & 7)) * 16);
        offa[ks] = wi * 32 * FA * kRowBytes + at;
        offb[ks] = wj * 32 * FB * kRowBytes + at;
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
    constexpr int NM = FA * FB, NR = FA + FB;
    constexpr int kSync = 1;  // MFMAs of a stage's last quarter in front of the barrier
    op_t a0[FA], b0[FB], a1[FA], b1[FB];
    // 16 k: the MFMAs on (ca, cb) and between them the LDS reads of the next 16 k, quarter KS of the stage at (imga, imgb).
    // KS == 0 means the last quarter of the stage before: first the barrier (the stage that follows has landed, at most `OUT`
    // instructions of later ones are on their way, and nobody reads this stage any more), then the DMA into its slots.
    // D0 ... D1: instructions of it that are issued here.
    auto kstep = [&](const op_t* ca, const op_t* cb, op_t* na, op_t* nb, const char* imga, const char* imgb, auto ks, auto reads, auto out,
                     auto d0, auto d1) {
        constexpr bool READS = decltype(reads)::value;
        constexpr int KS = decltype(ks)::value, OUT = decltype(out)::value, D0 = decltype(d0)::value, D1 = decltype(d1)::value;
        constexpr int R0 = KS == 0 && READS ? kSync + 1 : 0;  // MFMA behind which the reads begin
        constexpr int kPerSlot = (NR + NM - R0 - 1) / (NM - R0);
        constexpr int kDmaPerSlot = D1 > D0 ? (D1 - D0 + NM - R0 - 1) / (NM - R0) : 0;
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            mfma(acc[i / FB][i % FB], ca[i / FB], cb[i % FB]);
            if constexpr (KS == 0 && READS) {
                if (i == kSync) {
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(OUT) : "memory");
                    __builtin_amdgcn_s_barrier();
                }
            }
            if constexpr (READS) {
#pragma unroll
                for (int j = 0; j < kPerSlot; ++j) {
                    const int r = (i - R0) * kPerSlot + j;
                    if (i < R0 || r >= NR) continue;
                    if (r < FA) na[r] = read_op(imga, offa[KS] + r * 32 * kRowBytes);
                    else nb[r - FA] = read_op(imgb, offb[KS] + (r - FA) * 32 * kRowBytes);
                }
            }
            if constexpr (D1 > D0) {
#pragma unroll
                for (int j = 0; j < kDmaPerSlot; ++j) {
                    const int u = D0 + (i - R0) * kDmaPerSlot + j;
                    if (i >= R0 && u < D1) issue_one(u);
                }
            }
        }
    };
    using T = std::true_type;
    using F = std::false_type;
#define N_(v) std::integral_constant<int, (v)>{}
    auto slot_at = [&](int i) { return smem + (uint32_t)i % kSlots * kSlotBytes; };
    // A stage's DMA (x's of two stages on, W's of three) begins behind its barrier: kHead instructions of it in the last
    // quarter, the rest in the first of the next.  In front of the loop (there are at least three stages): both operands'
    // first, W's second, and the head of what the stage before the first would have begun.
    constexpr int kHead = (NDMA + 3) / 4, kTwo = (NDMA + 1) / 2, kThree = kTwo + kHead < NDMA ? kTwo + kHead : NDMA;
    issue_prepare(0, 0);
#pragma unroll
    for (int u = 0; u < NDMA; ++u) issue_one(u);
    issue_prepare(0, 1);
#pragma unroll
    for (int u = DB; u < NDMA; ++u) issue_one(u);
    issue_prepare(1, 2);
#pragma unroll
    for (int u = 0; u < kHead; ++u) issue_one(u);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(DA + kHead) : "memory");
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int m = 0; m < FA; ++m) a0[m] = read_op(slot_at(0), offa[0] + m * 32 * kRowBytes);
#pragma unroll
    for (int m = 0; m < FB; ++m) b0[m] = read_op(slot_at(1), offb[0] + m * 32 * kRowBytes);
    int st = 0;
    auto quarters = [&](auto more) {
        constexpr int M = decltype(more)::value;
        const char *ia = slot_at(2 * st), *ib = slot_at(2 * st + 1);
        kstep(a0, b0, a1, b1, ia, ib, N_(1), T{}, N_(0), N_(M * kHead), N_(M * kTwo));
        kstep(a1, b1, a0, b0, ia, ib, N_(2), T{}, N_(0), N_(M * kTwo), N_(M * kThree));
        kstep(a0, b0, a1, b1, ia, ib, N_(3), T{}, N_(0), N_(M * kThree), N_(M * NDMA));
    };
    for (; st + 3 < nst; ++st) {
        quarters(N_(1));
        issue_prepare(st + 2, st + 3);
        kstep(a1, b1, a0, b0, slot_at(2 * st + 2), slot_at(2 * st + 3), N_(0), T{}, N_(DA), N_(0), N_(kHead));
    }
    quarters(N_(1));
    issue_prepare(st + 2, st + 2);
    kstep(a1, b1, a0, b0, slot_at(2 * st + 2), slot_at(2 * st + 3), N_(0), T{}, N_(DA), N_(0), N_(DB));  // x's only
    ++st;
    quarters(N_(0));
    kstep(a1, b1, a0, b0, slot_at(2 * st + 2), slot_at(2 * st + 3), N_(0), T{}, N_(0), N_(0), N_(0));
    ++st;
    quarters(N_(0));
    kstep(a1, b1, a0, b0, smem, smem, N_(0), F{}, N_(0), N_(0), N_(0));
#undef N_
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");  // the last MFMAs leave the pipe before the read-out

    const uint32_t cols = gated ? 16 * FA : 32 * FA;  // of y, a wave's
    store_tile<DT, FA, FB>(g.ep, acc, (float*)smem + wave * kTileFloats<FA>, first + wj * 32 * FB, last, col0 + wi * cols, lane);
}

template <int DT, int WI, int WJ, int FA, int FB>
int dense_tiles(const DenseArgs& a, hipStream_t s) {
    static OncePerDevice once;
    constexpr int PA = 32 * WI * FA, PB = 32 * WJ * FB, kStageLds = kSlots * PA * kRowBytes;
    constexpr int kTileLds = WI * WJ * kTileFloats<FA> * 4;  // the epilogue's floats take the stages' place
    constexpr int kLds = kStageLds > kTileLds ? kStageLds : kTileLds;
    const bool opted_in = once.run([&] {
        return hipFuncSetAttribute((const void*)k_gemm_nt<DT, WI, WJ, FA, FB>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds) == hipSuccess;
    });
    if (!opted_in) return lds_refused(kLds);
    const bool gated = a.ep.act == kActSwiglu;
    const int64_t width = gated ? a.ep.n / 2 : a.ep.n, per = gated ? PA / 2 : PA, pb = PB;
    const int64_t tiles_n = (width + per - 1) / per;
    // ragged groups: each may end inside a tile
    const int64_t groups = a.rows.offsets ? (a.rows.experts < a.rows.rows ? a.rows.experts : a.rows.rows) : 1;
    const int64_t tiles_m = a.rows.offsets ? a.rows.rows / pb + groups : (a.rows.rows + pb - 1) / pb;
    const int64_t blocks = (tiles_n * tiles_m + 7) / 8 * 8;
    if (blocks > 0x7fffffff) {
        set_error("linear: too many tiles");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    hipLaunchKernelGGL((k_gemm_nt<DT, WI, WJ, FA, FB>), dim3((unsigned)blocks), dim3(64 * WI * WJ), kLds, s, a, (uint32_t)tiles_m, (uint32_t)tiles_n);
    return launch_status("linear");
}

bool dense_reaches(int64_t n, int64_t k, int64_t ldx, int64_t sources, bool gated, bool gathered) {
    constexpr int64_t kMost = (int64_t)0xffff0000;
    return (gated ? n : 512) * k * 2 < kMost && (gathered ? sources : 512) * ldx * 2 < kMost;
}

// 256 x 256 tiles by eight waves (1.29 to 1.38 PFLOP/s on 4096 x 28672 x 8192, by the card; one block per compute unit) or
// 128 x 128 by four (1.10, two blocks): whichever needs less time in rounds of blocks, a round of the small ones costing 0.6 of one of the large ones
// (4096 x 4096 x 4096: one round of large tiles 108 us, two of small ones 125; 2047 rows: 68 us in 512 small ones, 83 in 128
// large ones, half a round).
template <int DT>
int dense_typed(const DenseArgs& a, hipStream_t s) {
    const int64_t width = a.ep.n, groups = a.rows.offsets ? a.rows.experts : 1;
    auto rounds = [&](int64_t tile, int64_t at_once) {
        const int64_t rows = (a.rows.rows + tile - 1) / tile + (groups - 1) / 2;  // ragged groups: half a tile each on average
        return ((width + tile - 1) / tile * rows + at_once - 1) / at_once;
    };
    if (5 * rounds(256, 256) <= 3 * rounds(128, 512)) return dense_tiles<DT, 2, 4, 4, 2>(a, s);
    return dense_tiles<DT, 2, 2, 2, 2>(a, s);
}

int dense_launch(int dtype, const DenseArgs& a, hipStream_t s) {
    return dtype == NNCF_AMD_BF16 ? dense_typed<NNCF_AMD_BF16>(a, s) : dense_typed<NNCF_AMD_F16>(a, s);
}

}  // namespace wc
