// wc_gemm_codes.hip -- y = act(x W^T + bias) + residual for some tens to some hundreds of rows per group, W as it is stored:
// rows enough to fill matrix tiles, not enough to repay a decompressed copy of the weight in memory (wc_gemm_nt.hip takes over
// there, wc_linear_few.hip below).
//
// A block owns 128 rows of W by 128 FB rows of x (FB 1 or 2): 2 x 4 waves, each 2 x FB accumulators of v_mfma_f32_32x32x16, in
// stages of 64 k.  x goes global -> LDS by DMA as in the dense product (three slots).  W's codes, scales and zero points go
// into LDS the same way, four slots of each, every wave the 16 rows that its own lanes decompress: lane 4 r + q takes the 16
// codes 16 q ... of row r in each stage and writes their values into one of two slots of W tiles, eight at a time between the
// matrix instructions of the stage before.  No load in the loop has a register for its target, and one count of outstanding
// DMA per stage is all the waiting there is: codes arrive three stages after they are asked for, x two.
//
// A stage takes 1.1 us (FB 2; 0.85 FB 1) of the 0.5 that its matrix instructions need at 2 GHz: per stage and wave the LDS reads
// of the fragments, 75 vector and some 40 scalar instructions and a barrier stand one behind the other, and two waves per SIMD
// hide half of that (with four, half the work each, the sum was the same: 172 and 186 us for 256 rows of 28672 x 8192; asking
// for the next fragments before multiplying the last and counting slots instead of dividing gave 146).  Deeper rings change
// nothing.  256 rows of 28672 x 8192 int4: 145 us against 284 by strips and 278 densely; 97 of 4096 x 14336 NF4: 39 against 62
// and 151; 2000 rows over eight of 4096 x 14336 int4: 437 against 631 and 591.
//
// Where the tiles of y are fewer than the compute units, blocks share k: fp32 sums in the workspace, joined by join_sums.
#include "wc_gemm.h"

namespace wc {

constexpr int WI = 2, WJ = 4, NW = WI * WJ, FA = 2, kPA = 32 * WI * FA;  // waves; a wave's 32 rows of W; a block's rows of W

// a scale or zero point per lane, as DMA: an element of 1 or 2 bytes becomes a dword of LDS at lds + 4 lane
template <int BYTES>
__device__ __forceinline__ void dma_one(const i32x4& rsrc, uint32_t voff, uint32_t soff, uint32_t lds) {
    if constexpr (BYTES == 2)
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_ushort %0, %1, %2 offen lds" : : "v"(voff), "s"(rsrc), "s"(soff), "s"(lds) : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_ubyte %0, %1, %2 offen lds" : : "v"(voff), "s"(rsrc), "s"(soff), "s"(lds) : "memory", "m0");
}

template <int MODE, int FB>
struct CodesLds {
    static constexpr int PB = 32 * WJ * FB;
    static constexpr bool kFour = four_bit(MODE), kZero = MODE == NNCF_AMD_INT4_ASYM || MODE == NNCF_AMD_INT8_ASYM;
    static constexpr int kX = PB * kRowBytes, kW = kPA * kRowBytes, kRows = kPA / NW, kCodes = kRows * (kFour ? 32 : 64),
                         kPars = kRows * 2 * 4;  // per wave: W's rows, bytes of their codes, of scales (two a row: groups of 32)
    static constexpr int at_w = 3 * kX, at_codes = at_w + 2 * kW, at_scale = at_codes + 4 * NW * kCodes, at_zero = at_scale + 4 * NW * kPars,
                         end = at_zero + (kZero ? 4 * NW * kPars : 0);
    static constexpr int tile = NW * kTileFloats<FA> * 4, total = end > tile ? end : tile;
};

template <int MODE, int DT, int FB>
__global__ __launch_bounds__(64 * WI * WJ) void k_gemm_codes(CodesArgs g, uint32_t tiles_m, uint32_t tiles_n, uint32_t per) {
    using L = CodesLds<MODE, FB>;
    constexpr int PB = L::PB, DB = PB / (8 * NW), NC = L::kZero ? 3 : 2, NV = DB + NC;  // DMA instructions per wave and stage
    extern __shared__ __align__(16) char smem[];
    h2* lut = nullptr;
    if constexpr (MODE == NNCF_AMD_NF4) {
        __shared__ h2 pairs[kNf4Pairs];
        lut = pairs;
        fill_nf4<MODE>(lut);
    }
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t wi = wave / WJ, wj = wave % WJ;

    const bool gated = g.ep.act == kActSwiglu, halves = gated && g.kz == 1;  // halves: gate and other rows side by side in the tile
    const int64_t n = g.ep.n, width = halves ? n / 2 : n;
    if (g.rows.offsets) {
        if (blockIdx.x < tiles_n * tiles_m)  // (the gated tile's columns of y: half as many, in either form)
            zero_rows<64 * NW>(g.rows, g.ep, blockIdx.x % tiles_n, blockIdx.x / tiles_n, tiles_m, gated ? kPA / 2 : kPA);
        tiles_m = count_tiles<PB>(g.rows, tiles_m);
    }
    // a run of consecutive tiles per XCD (see the dense product), the row tile fastest, then the part of k: what shares W's rows
    // or x's columns runs side by side
    const uint32_t total = tiles_m * tiles_n * g.kz, each = (total + 7) / 8;
    const uint32_t id = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= each || id >= total) return;
    const uint32_t tm = id % tiles_m, z = id / tiles_m % g.kz, tn = id / tiles_m / g.kz;
    int expert;
    int64_t first, last;
    if (!find_tile<PB>(g.rows, tm, expert, first, last)) return;
    first = uniform(first), last = uniform(last);

    const int64_t col0 = (int64_t)tn * (halves ? kPA / 2 : kPA);
    const int st0 = (int)(z * per), all = (int)(g.k / 64), nst = all - st0 < (int)per ? all - st0 : (int)per;

    // x: as in the dense product
    const int64_t xorg = g.rows.slots ? 0 : first;
    const i32x4 rx = uniform(buffer_of((const char*)g.x + xorg * g.ldx * 2));
    uint32_t voff[DB], dst[DB];
#pragma unroll
    for (int u = 0; u < DB; ++u) {
        const uint32_t at8 = (u * NW + wave) * 8, row = at8 + (lane >> 3);
        int64_t r = first + row;
        r = r < last ? r : last - 1;
        voff[u] = (uint32_t)((source_row(g.rows, r) - xorg) * g.ldx * 2) + ((lane & 7) ^ (row >> 1 & 7)) * 16;
        dst[u] = at8 * kRowBytes;
    }
    // W: the row of the weight that row `t` of the tile holds, behind the expert's first
    auto weight_row = [&](uint32_t t) {
        int64_t c;
        if (halves) {
            constexpr uint32_t kHalf = 16 * FA;
            c = col0 + t / (2 * kHalf) * kHalf + t % kHalf;
            c = (c < width ? c : width - 1) + (t % (2 * kHalf) >= kHalf ? width : 0);
        } else {
            c = col0 + t;
            c = c < width ? c : width - 1;
        }
        return c;
    };
    constexpr uint32_t kRowPart = L::kFour ? 32 : 64;  // bytes of a row's codes in a stage
    const int64_t worg = halves ? 0 : col0, row_bytes = L::kFour ? g.k / 2 : g.k, w0 = (int64_t)expert * n + worg;
    const i32x4 rc = uniform(buffer_of(g.codes + w0 * row_bytes));
    constexpr uint32_t kRows = L::kRows, kAsk = L::kCodes / 16, kOf = 64 / kRows;  // lanes that ask for codes; lanes per row
    const uint32_t asked = lane % kAsk * 16;
    const uint32_t voff_c = (uint32_t)((weight_row(wave * kRows + asked / kRowPart) - worg) * row_bytes) + asked % kRowPart;
    const uint32_t share = lane % kOf, trow = wave * kRows + lane / kOf;
    // first groups: of the row that a lane asks parameters for (two lanes a row), of the one that it decompresses
    const uint32_t pask = (uint32_t)(weight_row(wave * kRows + lane / 2 % kRows) - worg) * g.groups;
    const uint32_t prow = (uint32_t)(weight_row(trow) - worg) * g.groups;
    constexpr int SB = MODE == NNCF_AMD_MXFP4 ? 1 : 2;
    const i32x4 rs = uniform(buffer_of((const char*)g.scale + w0 * g.groups * SB));
    const int64_t z_first = w0 * g.groups;
    const uint32_t z_odd = MODE == NNCF_AMD_INT4_ASYM ? (uint32_t)(z_first & 1) : 0;
    const i32x4 rz = uniform(buffer_of(L::kZero ? g.zp + (MODE == NNCF_AMD_INT4_ASYM ? z_first >> 1 : z_first) : g.codes));
    // the group of a stage's 16 codes: `group_stages` stages each, or (groups of 32) two in a stage
    auto group_of = [&](int st, uint32_t half) { return g.group_stages ? (uint32_t)((uint32_t)st * g.magic >> 32) : 2 * (uint32_t)st + half; };

    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)smem;
    // What is brought in next: x's stage and slot, the codes' stage with the offset of its groups.  Behind the last stage the last
    // is asked for again, so that the count of outstanding DMA stays the same; nobody reads it.
    int next_x = 0, next_c = 0, group_left = (int)g.group_stages - (g.group_stages ? st0 % (int)g.group_stages : 0);
    uint32_t so_x = (uint32_t)st0 * kRowBytes, so_c = (uint32_t)st0 * kRowPart, slot_x = 0;
    uint32_t gi = pask + group_of(st0, lane & 1);
    auto issue_x = [&] {
#pragma unroll
        for (int u = 0; u < DB; ++u) dma16(rx, voff[u], so_x, lds0 + slot_x + dst[u]);
        slot_x = slot_x == 2 * L::kX ? 0 : slot_x + L::kX;
        if (++next_x < nst) so_x += kRowBytes;
    };
    auto issue_codes = [&] {
        const uint32_t slot = ((uint32_t)next_c & 3) * NW + wave;
        if (lane < kAsk) dma16(rc, voff_c, so_c, lds0 + L::at_codes + slot * L::kCodes);
        if (lane < 2 * kRows) {
            dma_one<SB>(rs, gi * SB, 0, lds0 + L::at_scale + slot * L::kPars);
            if constexpr (MODE == NNCF_AMD_INT4_ASYM) dma_one<1>(rz, (gi + z_odd) >> 1, 0, lds0 + L::at_zero + slot * L::kPars);
            if constexpr (MODE == NNCF_AMD_INT8_ASYM) dma_one<1>(rz, gi, 0, lds0 + L::at_zero + slot * L::kPars);
        }
        if (++next_c < nst) {
            so_c += kRowPart;
            if (!g.group_stages) gi += 2;
            else if (--group_left == 0) gi += 1, group_left = (int)g.group_stages;
        }
    };
    // a stage's codes and parameters of this lane, and its values' way into the W slot, eight at a time
    constexpr int kEights = 8 / kOf, kWords = kEights * (L::kFour ? 1 : 2);
    struct Codes {
        uint32_t p[kWords], scale, zero;
    };
    char* const wdst = smem + L::at_w + trow * kRowBytes;
    const uint32_t from_c = L::at_codes + wave * L::kCodes + lane * (L::kCodes / 64);
    const uint32_t from_p = L::at_scale + wave * L::kPars + (lane / kOf * 2 + share / (kOf / 2)) * 4;
    auto read_codes = [&](int st) {
        Codes c{};
        const char *at = smem + from_c + ((uint32_t)st & 3) * NW * L::kCodes, *par = smem + from_p + ((uint32_t)st & 3) * NW * L::kPars;
        __builtin_memcpy(c.p, __builtin_assume_aligned(at, 4 * kWords), 4 * kWords);
        c.scale = *(const uint32_t*)par;
        if constexpr (L::kZero) c.zero = *(const uint32_t*)(par + (L::at_zero - L::at_scale));
        if constexpr (MODE == NNCF_AMD_INT4_ASYM)
            c.zero = c.zero >> (4 * ((prow + group_of((st < nst ? st : nst - 1) + st0, share / (kOf / 2)) + z_odd) & 1)) & 15u;
        return c;
    };
    auto write_eight = [&](int st, const Codes& c, int i) {
        const GroupPar<MODE> par = par_of<MODE>(c.scale, c.zero);
        *(u32v4*)(wdst + ((uint32_t)st & 1) * L::kW + ((kEights * share + i) ^ (trow >> 1 & 7)) * 16) =
            L::kFour ? dequant8<MODE, DT>(c.p[i], 0, par, lut) : dequant8<MODE, DT>(c.p[2 * i % kWords], c.p[(2 * i + 1) % kWords], par, lut);
    };

    typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
    typedef _Float16 hf8 __attribute__((ext_vector_type(8)));
    auto mfma = [](const u32v4& a, const u32v4& b, const f32x16& c) {
        if constexpr (DT == NNCF_AMD_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, a), __builtin_bit_cast(bf8, b), c, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(hf8, a), __builtin_bit_cast(hf8, b), c, 0, 0, 0);
    };
    f32x16 acc[FA][FB];
#pragma unroll
    for (int a = 0; a < FA; ++a)
#pragma unroll
        for (int b = 0; b < FB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.0f;
    const uint32_t r32 = lane & 31, kh = lane >> 5;
    struct Frags {
        u32v4 a[FA], b[FB];
    };
    uint32_t off_a[4], off_b[4];  // 16 k each
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        const uint32_t at = r32 * kRowBytes + (((2 * ks + kh) ^ (r32 >> 1 & 7)) * 16);
        off_a[ks] = wi * FA * 32 * kRowBytes + at;
        off_b[ks] = wj * FB * 32 * kRowBytes + at;
    }
    auto read_frags = [&](const char* wimg, const char* ximg, int ks) {
        Frags f;
#pragma unroll
        for (int i = 0; i < FA; ++i) f.a[i] = *(const u32v4*)(wimg + off_a[ks] + i * 32 * kRowBytes);
#pragma unroll
        for (int i = 0; i < FB; ++i) f.b[i] = *(const u32v4*)(ximg + off_b[ks] + i * 32 * kRowBytes);
        return f;
    };
    auto multiply = [&](const Frags& f) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j) acc[i][j] = mfma(f.a[i], f.b[j], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    };

    issue_codes();
    issue_codes();
    issue_x();
    issue_codes();
    issue_x();
    issue_codes();
    __syncthreads();  // NF4's table
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NC + NV) : "memory");
    {
        const Codes c = read_codes(0);
#pragma unroll
        for (int i = 0; i < kEights; ++i) write_eight(0, c, i);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    uint32_t read_x = 0;
#pragma unroll 1
    for (int st = 0; st < nst; ++st) {
        const char *wimg = smem + L::at_w + ((uint32_t)st & 1) * L::kW, *ximg = smem + read_x;
        const Frags f0 = read_frags(wimg, ximg, 0);
        const Codes c = read_codes(st + 1);
        const Frags f1 = read_frags(wimg, ximg, 1);
        __builtin_amdgcn_sched_barrier(0);
        issue_x();
        multiply(f0);
        issue_codes();
        const Frags f2 = read_frags(wimg, ximg, 2);
        write_eight(st + 1, c, 0);
        multiply(f1);
        const Frags f3 = read_frags(wimg, ximg, 3);
        if constexpr (kEights > 1) write_eight(st + 1, c, 1);
        multiply(f2);
        multiply(f3);
        read_x = read_x == 2 * L::kX ? 0 : read_x + L::kX;
        // x of the next stage and the codes of the one after it have landed
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(NC + NV) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the DMA behind the last stage, before its LDS gets the sums

    Epilogue part = g.ep;
    if (g.kz > 1) part = Epilogue{nullptr, nullptr, g.sums + (int64_t)z * g.rows.rows * n, nullptr, 0, n, n, kActNone, 1, n % 4 == 0};
    store_tile<DT, FA, FB>(part, acc, (float*)smem + wave * kTileFloats<FA>, first + wj * 32 * FB, last, col0 + wi * (halves ? 16 : 32) * FA, lane);
}

template <int MODE, int DT, int FB>
int codes_tiles(const CodesArgs& a, hipStream_t s) {
    static OncePerDevice once;
    constexpr int kLds = CodesLds<MODE, FB>::total, PB = 32 * WJ * FB;
    static_assert(kLds + (MODE == NNCF_AMD_NF4 ? 4 * kNf4Pairs : 0) <= 160 * 1024, "LDS of a compute unit");
    const bool opted_in = once.run([&] {
        return hipFuncSetAttribute((const void*)k_gemm_codes<MODE, DT, FB>, hipFuncAttributeMaxDynamicSharedMemorySize, kLds) == hipSuccess;
    });
    if (!opted_in) return lds_refused(kLds);
    const bool halves = a.ep.act == kActSwiglu && a.kz == 1;
    const int64_t tiles_n = ((halves ? a.ep.n / 2 : a.ep.n) + (halves ? 63 : 127)) / (halves ? 64 : 128);
    const int64_t groups = a.rows.offsets ? (a.rows.experts < a.rows.rows ? a.rows.experts : a.rows.rows) : 1;
    const int64_t tiles_m = a.rows.offsets ? a.rows.rows / PB + groups : (a.rows.rows + PB - 1) / PB;
    const int64_t blocks = (tiles_n * tiles_m * a.kz + 7) / 8 * 8;
    if (blocks > 0x7fffffff) {
        set_error("linear: too many tiles");
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    const int64_t stages = a.k / 64, per = (stages + a.kz - 1) / a.kz;
    hipLaunchKernelGGL((k_gemm_codes<MODE, DT, FB>), dim3((unsigned)blocks), dim3(64 * WI * WJ), kLds, s, a, (uint32_t)tiles_m, (uint32_t)tiles_n, (uint32_t)per);
    const int st = launch_status("linear");
    return st != NNCF_AMD_OK || a.kz == 1 ? st : join_sums(DT, a.sums, a.kz, a.rows, a.ep, s);
}

template <int DT>
int codes_typed(int mode, int fb, const CodesArgs& a, hipStream_t s) {
#define CODES(M) \
    case M: return fb == 1 ? codes_tiles<M, DT, 1>(a, s) : codes_tiles<M, DT, 2>(a, s);
    switch (mode) {
        CODES(NNCF_AMD_INT4_ASYM)
        CODES(NNCF_AMD_INT4_SYM)
        CODES(NNCF_AMD_NF4)
        CODES(NNCF_AMD_MXFP4)
        case NNCF_AMD_INT8_ASYM: return codes_tiles<NNCF_AMD_INT8_ASYM, DT, 1>(a, s);
        default: return codes_tiles<NNCF_AMD_INT8_SYM, DT, 1>(a, s);
    }
#undef CODES
}
int codes_launch(int dtype, int mode, int fb, const CodesArgs& a, hipStream_t s) {
    return dtype == NNCF_AMD_BF16 ? codes_typed<NNCF_AMD_BF16>(mode, fb, a, s) : codes_typed<NNCF_AMD_F16>(mode, fb, a, s);
}

bool codes_fits(int mode, int64_t n, int64_t k, int64_t gs, const void* codes) {
    // (the multiplier that divides stages by a group's is exact below 2^16 of them)
    return k % 64 == 0 && k <= (1 << 20) && (gs == k || gs % 64 == 0 || gs == 32) && ((uintptr_t)codes & 15) == 0 && mode <= NNCF_AMD_MXFP4 &&
           n * k < ((int64_t)1 << 31);
}

// The shape with the least time: rounds of blocks on the 256 compute units, a stage of 64 k `kStage` us each and 6 for a round's
// start and end, the join of shared k its launch and its bytes.
CodesShape codes_plan(int mode, int64_t n, int64_t k, bool gated, int64_t rows, int64_t experts, bool grouped) {
    constexpr double kStage[2] = {0.85, 1.1};
    CodesShape best{1, 1, 1e30};
    const int64_t stages = k / 64;
    for (int fb = 1; fb <= (four_bit(mode) ? 2 : 1); ++fb) {
        const int64_t tiles_m = (rows + 128 * fb - 1) / (128 * fb) + (grouped ? (experts - 1) / 2 : 0);
        for (int64_t kz = 1; kz <= 16 && kz * 4 <= stages; ++kz) {
            const int64_t per = (stages + kz - 1) / kz;
            if ((stages + per - 1) / per != kz) continue;  // some would have none
            const int64_t tiles_n = gated && kz == 1 ? (n / 2 + 63) / 64 : (n + 127) / 128;
            const double rounds = (double)((tiles_n * tiles_m * kz + 255) / 256);
            double us = rounds * ((double)per * kStage[fb - 1] + 6.0);
            if (kz > 1) us += 3.0 + (double)(kz * rows * n) * 8.0 / 4.0e6;
            if (us < best.us) best = CodesShape{fb, (int)kz, us};
        }
    }
    return best;
}

}  // namespace wc
