// wc_experts.hip -- routing of tokens to experts, and the weighted sum of the experts' answers.
//
// Route: a token's top-k experts by falling logit (ties: the lower number first; a NaN ranks below every number), their
// softmax weights in fp32 -- over the chosen ones (renormalised) or over all experts --, and the plan that the grouped
// products run by: slots (token * topk + place) in the order of their experts, stable, so that the rows of expert e are
// [offsets[e], offsets[e + 1]); rows[slot] is a slot's place in that order, slots[row] its inverse.  Masked tokens (padding)
// have experts and rows -1, weights 0, and no place; the rows behind the last have slots -1.
// A row of logits that are all -inf leaves nothing to choose: its weights are 0 (its experts the first ones).
#include "wc_linear.h"

namespace wc {

constexpr int kRouteThreads = 512;
constexpr int kRouteWaves = kRouteThreads / 64;
constexpr int kRouteSlots = 4096;      // slots of one block: their experts and ranks are held in LDS
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopk = 64;
constexpr int kRouteBlocks = 256;      // blocks that the tokens are dealt over while the slots of a block fit

template <int DT>
__device__ __forceinline__ float logit(const void* p, int64_t i) { return Elem<DT>::load(p, i); }

// a float's order as an integer: NaN lowest (0), then -inf ... +inf; -0 and +0 are equal
__device__ __forceinline__ uint32_t order_of(float v) {
    if (v != v) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, v + 0.0f);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
    if (o == 0) return __builtin_nanf("");
    return __builtin_bit_cast(float, (o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int d) {
    return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), d, 64) << 32) | (uint32_t)__shfl_xor((int)v, d, 64);
}

// maximum over aligned sets of G lanes: inside 16 lanes by DPP (a shuffle goes through LDS), above that by shuffles
template <int CTRL>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xf, 0xf, true);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, true);
    return (uint64_t)hi << 32 | lo;
}
template <int G>
__device__ __forceinline__ uint64_t max_over(uint64_t v) {
    auto larger = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
    if constexpr (G >= 2) v = larger(v, dpp64<0xB1>(v));    // quad_perm [1,0,3,2]
    if constexpr (G >= 4) v = larger(v, dpp64<0x4E>(v));    // quad_perm [2,3,0,1]
    if constexpr (G >= 8) v = larger(v, dpp64<0x141>(v));   // row_half_mirror
    if constexpr (G >= 16) v = larger(v, dpp64<0x140>(v));  // row_mirror
    if constexpr (G >= 32) v = larger(v, shfl_xor64(v, 16));
    if constexpr (G >= 64) v = larger(v, shfl_xor64(v, 32));
    return v;
}

struct RouteArgs {
    const void* logits;
    int64_t ldl, tokens;
    int experts, topk, renormalize, blocks;
    int64_t per_block;  // tokens
    const uint8_t* mask;
    float* weights;
    int32_t *ids, *rows, *slots, *offsets;
    int32_t* hist;  // [experts][blocks] (more than one block)
};

// G lanes share a token, each holds V of its logits.  topk rounds of a maximum over the lanes on (order, lowest expert) keys:
// the chosen key is cleared where it was found.  Then the block's slots are ranked among those of the same expert: a wave
// takes 64 consecutive slots at a time and compares expert numbers bit by bit with ballots, so that the order is stable and
// no atomic decides it.  Bound by latency (32000 tokens over 64 experts read 4 MB): 18 us for six experts each, 4.2 us for four
// tokens over eight.
template <int DT, int G, int V>
__global__ __launch_bounds__(kRouteThreads) void k_route(RouteArgs a) {
    __shared__ float sel[kRouteSlots];
    __shared__ int16_t ids[kRouteSlots];
    __shared__ uint16_t rank[kRouteSlots];
    __shared__ uint16_t hist[kRouteWaves][kRouteMaxExperts];  // up to kRouteSlots
    __shared__ int32_t start[kRouteMaxExperts + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int gl = tid & (G - 1), slot_of_group = tid / G;
    constexpr int TB = kRouteThreads / G;
    const int64_t t0 = (int64_t)blockIdx.x * a.per_block;
    const int64_t t1 = t0 + a.per_block < a.tokens ? t0 + a.per_block : a.tokens;
    const int count = t1 > t0 ? (int)(t1 - t0) : 0;
    for (int base = 0; base < count; base += TB) {
        const int local = base + slot_of_group;
        const bool live = local < count;
        const int64_t t = t0 + (live ? local : 0);
        const bool masked = a.mask && !a.mask[t];
        uint64_t key[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = i * G + gl;
            key[i] = e < a.experts ? ((uint64_t)order_of(logit<DT>(a.logits, t * a.ldl + e)) << 32) | (0xffffffffu - (uint32_t)e) : 0;
        }
        bool nan = false;
#pragma unroll
        for (int i = 0; i < V; ++i) nan = nan || (key[i] != 0 && (key[i] >> 32) == 0);
        float top = 0.0f, all = 0.0f, chosen = 0.0f;
        float* mine = sel + slot_of_group * a.topk;
        for (int j = 0; j < a.topk; ++j) {
            uint64_t best = key[0];
#pragma unroll
            for (int i = 1; i < V; ++i) best = key[i] > best ? key[i] : best;
            best = max_over<G>(best);
            const float v = value_of((uint32_t)(best >> 32));
            if (j == 0) {
                top = v;
                if (!a.renormalize) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        if (key[i]) all += expf(value_of((uint32_t)(key[i] >> 32)) - top);
                    all = lanes_allreduce<G>(all, OpAdd());
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) key[i] = key[i] == best ? 0 : key[i];
            const float w = expf(v - top);
            chosen += w;
            if (gl == 0 && live) {
                const int e = (int)(0xffffffffu - (uint32_t)best);
                mine[j] = w;
                ids[local * a.topk + j] = masked ? (int16_t)-1 : (int16_t)e;
                a.ids[t * a.topk + j] = masked ? -1 : e;
            }
        }
        const bool any_nan = max_over<G>(nan) != 0;
        if (gl == 0 && live) {
            const float total = a.renormalize ? chosen : all;
            const bool none = masked || (top == -__builtin_inff() && !any_nan);
            for (int j = 0; j < a.topk; ++j) a.weights[t * a.topk + j] = none ? 0.0f : mine[j] / total;
        }
    }
    for (int i = tid; i < kRouteWaves * a.experts; i += kRouteThreads) hist[i / a.experts][i % a.experts] = 0;
    __syncthreads();
    const int n = count * a.topk;
    const int per_wave = ((n + kRouteWaves - 1) / kRouteWaves + 63) & ~63;
    const int bits = 32 - __clz(a.experts);  // of the largest number that stands for "none"
    volatile uint16_t* counts = hist[wave];  // lanes of one wave read what others have written a round before
    for (int s = wave * per_wave; s < n && s < (wave + 1) * per_wave; s += 64) {
        const bool in = s + lane < n;
        const int e = in ? ids[s + lane] : -1;
        const uint32_t v = e < 0 ? (uint32_t)a.experts : (uint32_t)e;
        uint64_t same = ~0ull;
        for (int b = 0; b < bits; ++b) {
            const uint64_t m = __ballot((v >> b) & 1);
            same &= ((v >> b) & 1) ? m : ~m;
        }
        if (e >= 0) {
            const int before = __popcll(same & ((1ull << lane) - 1));
            const int sofar = counts[e];
            rank[s + lane] = (uint16_t)(sofar + before);
            // the last lane of an expert's set adds the set; the others have read the count (one wave: in order)
            if ((same >> lane) == 1ull) counts[e] = (uint16_t)(sofar + before + 1);
        }
    }
    __syncthreads();
    for (int e = tid; e < a.experts; e += kRouteThreads) {  // exclusive over the waves; the total to `start`
        int32_t sum = 0;
        for (int w = 0; w < kRouteWaves; ++w) {
            const int32_t c = hist[w][e];
            hist[w][e] = (uint16_t)sum;
            sum += c;
        }
        start[e] = sum;
        if (a.blocks > 1) a.hist[(int64_t)e * a.blocks + blockIdx.x] = sum;
    }
    __syncthreads();
    if (a.blocks == 1 && wave == 0) {  // exclusive over the experts
        int32_t carry = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int32_t c = e0 + lane < a.experts ? start[e0 + lane] : 0;
            int32_t sum = c;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int32_t u = __shfl_up(sum, d, 64);
                if (lane >= d) sum += u;
            }
            if (e0 + lane < a.experts) {
                start[e0 + lane] = carry + sum - c;
                a.offsets[e0 + lane] = carry + sum - c;
            }
            carry += __shfl(sum, 63, 64);
        }
        if (lane == 0) start[a.experts] = carry, a.offsets[a.experts] = carry;
    }
    __syncthreads();
    for (int s = tid; s < n; s += kRouteThreads) {
        const int e = ids[s];
        const int64_t slot = t0 * a.topk + s;
        if (a.blocks == 1) {
            const int row = e < 0 ? -1 : start[e] + hist[s / per_wave][e] + rank[s];
            a.rows[slot] = row;
            if (row >= 0) a.slots[row] = s;
            if (s >= start[a.experts]) a.slots[s] = -1;
        } else {
            a.rows[slot] = e < 0 ? -1 : hist[s / per_wave][e] + rank[s];  // in the block; k_route_place adds the rest
        }
    }
}

// Adds what stands before the block: the experts of lower number, and the same expert in earlier blocks.  Every block sums the
// counts it needs by itself (experts x blocks numbers from the L2) instead of a launch in between.  Latency again: 13 us for
// 192000 slots.
__global__ __launch_bounds__(kRouteThreads) void k_route_place(RouteArgs a) {
    __shared__ int32_t start[kRouteMaxExperts + 1], before[kRouteMaxExperts];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int e = wave; e < a.experts; e += kRouteWaves) {
        int32_t all = 0, mine = 0;
        for (int b = lane; b < a.blocks; b += 64) {
            const int32_t c = a.hist[(int64_t)e * a.blocks + b];
            all += c;
            if (b < (int)blockIdx.x) mine += c;
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            all += __shfl_xor(all, d, 64);
            mine += __shfl_xor(mine, d, 64);
        }
        if (lane == 0) start[e] = all, before[e] = mine;
    }
    __syncthreads();
    if (wave == 0) {
        int32_t carry = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 64) {
            const int32_t c = e0 + lane < a.experts ? start[e0 + lane] : 0;
            int32_t sum = c;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int32_t u = __shfl_up(sum, d, 64);
                if (lane >= d) sum += u;
            }
            if (e0 + lane < a.experts) start[e0 + lane] = carry + sum - c;
            carry += __shfl(sum, 63, 64);
        }
        if (lane == 0) start[a.experts] = carry;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = tid; e <= a.experts; e += kRouteThreads) a.offsets[e] = start[e];
    const int64_t s0 = (int64_t)blockIdx.x * a.per_block * a.topk;
    int64_t s1 = s0 + a.per_block * a.topk;
    if (s1 > a.tokens * a.topk) s1 = a.tokens * a.topk;
    for (int64_t s = s0 + tid; s < s1; s += kRouteThreads) {
        const int e = a.ids[s];
        if (e >= 0) {
            const int row = start[e] + before[e] + a.rows[s];
            a.rows[s] = row;
            a.slots[row] = (int32_t)s;
        }
        if (s >= start[a.experts]) a.slots[s] = -1;
    }
}

// d logits from d weights.  With w the weights, p the softmax over all experts, D = sum_j w_j dw_j:
//     renormalised:  w_i (dw_i - D) for the chosen i, 0 elsewhere;      else:  [i chosen] w_i dw_i - p_i D
template <int DT, int G, int V>
__global__ __launch_bounds__(256) void k_route_grad(const void* __restrict__ logits, int64_t ldl, int64_t tokens, int experts, int topk,
                                                    int renormalize, const float* __restrict__ weights, const int32_t* __restrict__ ids,
                                                    const float* __restrict__ dweights, void* __restrict__ dlogits) {
    const int64_t t = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const int gl = threadIdx.x & (G - 1);
    const bool live = t < tokens;
    const int64_t tt = live ? t : 0;
    float x[V], p[V];
    float top = -__builtin_inff(), all = 0.0f, dot = 0.0f;
    const bool none = ids[tt * topk] < 0;
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = p[i] = 0.0f;
    if (!renormalize) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int e = i * G + gl;
            x[i] = e < experts ? logit<DT>(logits, tt * ldl + e) : -__builtin_inff();
            top = fmaxf(top, x[i]);
        }
        top = lanes_allreduce<G>(top, OpMax());
        const bool empty = top == -__builtin_inff();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            p[i] = i * G + gl < experts && !empty ? expf(x[i] - top) : 0.0f;
            all += p[i];
        }
        all = lanes_allreduce<G>(all, OpAdd());
        if (empty) all = 1.0f;
    }
    for (int j = 0; j < topk; ++j) dot += weights[tt * topk + j] * dweights[tt * topk + j];
    float g[V];
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = renormalize ? 0.0f : -(p[i] / all) * dot;
    for (int j = 0; j < topk; ++j) {
        const int e = ids[tt * topk + j];
        const float w = weights[tt * topk + j], v = w * (dweights[tt * topk + j] - (renormalize ? dot : 0.0f));
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i * G + gl == e) g[i] += v;
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int e = i * G + gl;
        if (e >= experts) break;
        const float v = none ? 0.0f : g[i];
        if constexpr (DT == NNCF_AMD_F32) ((float*)dlogits)[t * experts + e] = v;
        else ((uint16_t*)dlogits)[t * experts + e] = from_f32<DT>(v);
    }
}

// ------------------------------------------------------------------------------------------------------------- weighted sum
// out[t] = sum_j w[t, j] y[rows[t, j]] in fp32, rounded once (weights == nullptr: plain sum).  A gather: every answer is read
// once and in the order j = 0 ... topk - 1, so the result does not depend on the schedule.  Bound by the bytes of y: 16000
// tokens of two rows of 4096 in 79 us, 5.0 TB/s.
// VEC: columns per thread; threads in x run along the columns, in y over tokens.
template <int IN, int OUT, int VEC>
__global__ __launch_bounds__(256) void k_combine(const void* __restrict__ y, int64_t ldy, int64_t total_rows, const float* __restrict__ weights,
                                                 const int32_t* __restrict__ rows, int64_t tokens, int topk, int64_t n,
                                                 uint16_t* __restrict__ out) {
    const int64_t t = (int64_t)blockIdx.y * blockDim.y + threadIdx.y;
    const int64_t c = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * VEC;
    if (t >= tokens || c >= n) return;
    float s[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) s[i] = 0.0f;
#pragma unroll 4
    for (int j = 0; j < topk; ++j) {
        const int32_t r = rows[t * topk + j];
        if (r < 0 || r >= total_rows) continue;
        const float w = weights ? weights[t * topk + j] : 1.0f;
        if constexpr (VEC == 8) {
            float v[8];
            if constexpr (IN == NNCF_AMD_F32) {
                unpack<IN>(*(const Vec16*)((const float*)y + r * ldy + c), v);
                unpack<IN>(*(const Vec16*)((const float*)y + r * ldy + c + 4), v + 4);
            } else {
                unpack<IN>(*(const Vec16*)((const uint16_t*)y + r * ldy + c), v);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += w * v[i];
        } else {
            s[0] += w * Elem<IN>::load(y, r * ldy + c);
        }
    }
    if constexpr (VEC == 8)
        *(u32v4*)(out + t * n + c) = u32v4{pair_of<OUT>(s[0], s[1]), pair_of<OUT>(s[2], s[3]), pair_of<OUT>(s[4], s[5]), pair_of<OUT>(s[6], s[7])};
    else
        out[t * n + c] = from_f32<OUT>(s[0]);
}

// dy[rows[s]] = w[s] dout[t],  dw[s] = <dout[t], y[rows[s]]>: a wave per slot; the rows without a slot get zeros.  The bytes of
// y, dout and dy: 126 us for the same, 5.2 TB/s.
template <int DT, int VEC>
__global__ __launch_bounds__(256) void k_combine_grad(const uint16_t* __restrict__ dout, const uint16_t* __restrict__ y, int64_t ldy,
                                                      const float* __restrict__ weights, const int32_t* __restrict__ rows,
                                                      const int32_t* __restrict__ slots, int64_t total, int topk, int64_t n,
                                                      uint16_t* __restrict__ dy, float* __restrict__ dweights) {
    const int64_t s = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (s >= total) return;
    const int32_t r = rows[s];
    const bool here = r >= 0 && r < total;
    if (dy && slots[s] < 0)  // row s has no slot
        for (int64_t c = lane; c < n; c += 64) dy[s * n + c] = 0;
    float dot = 0.0f;
    if (here) {
        const float w = weights[s];
        const uint16_t* d = dout + (s / topk) * n;
        const uint16_t* yr = y + r * ldy;
        uint16_t* o = dy ? dy + r * n : nullptr;
        for (int64_t c = (int64_t)lane * VEC; c < n; c += 64 * VEC) {
            if constexpr (VEC == 8) {
                float a[8];
                unpack<DT>(*(const Vec16*)(d + c), a);
                if (dweights) {
                    float b[8];
                    unpack<DT>(*(const Vec16*)(yr + c), b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) dot += a[i] * b[i];
                }
                if (o)
                    *(u32v4*)(o + c) = u32v4{pair_of<DT>(w * a[0], w * a[1]), pair_of<DT>(w * a[2], w * a[3]), pair_of<DT>(w * a[4], w * a[5]),
                                             pair_of<DT>(w * a[6], w * a[7])};
            } else {
                const float a = to_f32<DT>(d[c]);
                if (dweights) dot += a * to_f32<DT>(yr[c]);
                if (o) o[c] = from_f32<DT>(w * a);
            }
        }
    }
    if (dweights) {
        dot = lanes_allreduce<64>(dot, OpAdd());
        if (lane == 0) dweights[s] = dot;
    }
}

// ------------------------------------------------------------------------------------------------------------------- host
int check_route(const char* what, int dtype, int64_t tokens, int64_t experts, int64_t topk, int64_t ldl) {
    if (dtype != NNCF_AMD_F32 && dtype != NNCF_AMD_F16 && dtype != NNCF_AMD_BF16) {
        set_error("%s: logits are fp32, fp16 or bf16 (dtype %d)", what, dtype);
        return NNCF_AMD_ERR_DTYPE;
    }
    if (tokens < 0 || experts < 1 || topk < 1 || topk > experts || ldl < experts) {
        set_error("%s: bad shape (tokens=%lld experts=%lld topk=%lld)", what, (long long)tokens, (long long)experts, (long long)topk);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (experts > kRouteMaxExperts || topk > kRouteMaxTopk || tokens * topk > 0x7fffffff) {
        set_error("%s: up to %d experts, %d of them per token and 2^31 - 1 slots are supported", what, kRouteMaxExperts, kRouteMaxTopk);
        return NNCF_AMD_ERR_UNSUPPORTED;
    }
    return NNCF_AMD_OK;
}
int lanes_of(int64_t experts) { return experts <= 8 ? 1 : experts <= 32 ? 8 : experts <= 64 ? 16 : experts <= 128 ? 32 : 64; }
// Tokens per block.  Up to four passes of one block's lanes stay in one block (one launch); else about kRouteBlocks blocks.
int64_t tokens_per_block(int64_t tokens, int64_t experts, int64_t topk) {
    const int64_t pass = kRouteThreads / lanes_of(experts), fit = kRouteSlots / topk;
    if (tokens <= 4 * pass && tokens <= fit) return tokens > 0 ? tokens : 1;
    int64_t per = (tokens + kRouteBlocks - 1) / kRouteBlocks;
    per = (per + pass - 1) / pass * pass;
    return per < fit ? per : fit;
}

#define BY_EXPERTS(GO, DT)                           \
    if (experts <= 8) GO(DT, 1, 8);                  \
    else if (experts <= 32) GO(DT, 8, 4);            \
    else if (experts <= 64) GO(DT, 16, 4);           \
    else if (experts <= 128) GO(DT, 32, 4);          \
    else if (experts <= 256) GO(DT, 64, 4);          \
    else if (experts <= 512) GO(DT, 64, 8);          \
    else GO(DT, 64, 16);
#define BY_TYPE(GO)                                            \
    if (dtype == NNCF_AMD_F32) { BY_EXPERTS(GO, NNCF_AMD_F32) } \
    else if (dtype == NNCF_AMD_F16) { BY_EXPERTS(GO, NNCF_AMD_F16) } \
    else { BY_EXPERTS(GO, NNCF_AMD_BF16) }

}  // namespace wc

extern "C" size_t nncf_amd_route_experts_workspace(int64_t tokens, int64_t experts, int64_t topk) {
    using namespace wc;
    if (tokens < 1 || experts < 1 || topk < 1 || topk > kRouteMaxTopk) return 0;
    const int64_t per = tokens_per_block(tokens, experts, topk), blocks = (tokens + per - 1) / per;
    return blocks > 1 ? (size_t)(blocks * experts) * 4 : 0;
}

extern "C" int nncf_amd_route_experts(const void* logits, int dtype, int64_t ldl, int64_t tokens, int64_t experts, int64_t topk,
                                      int renormalize, const uint8_t* mask, float* weights, int32_t* ids, int32_t* rows, int32_t* slots,
                                      int32_t* offsets, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace wc;
    int st = check_route("route_experts", dtype, tokens, experts, topk, ldl);
    if (st != NNCF_AMD_OK) return st;
    if (!offsets || (tokens > 0 && (!logits || !weights || !ids || !rows || !slots))) {
        set_error("route_experts: null argument");
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const size_t need = nncf_amd_route_experts_workspace(tokens, experts, topk);
    if (need && (!workspace || workspace_bytes < need)) {
        set_error("route_experts: workspace of %zu bytes needed", need);
        return NNCF_AMD_ERR_WORKSPACE;
    }
    const int64_t per = tokens_per_block(tokens, experts, topk);
    const int64_t blocks = tokens > 0 ? (tokens + per - 1) / per : 1;  // no tokens: one block writes the offsets
    const RouteArgs a{logits, ldl, tokens, (int)experts, (int)topk, renormalize, (int)blocks, per, mask, weights, ids, rows, slots, offsets, (int32_t*)workspace};
    hipStream_t s = (hipStream_t)stream;
#define GO(DT, G, V) hipLaunchKernelGGL((k_route<DT, G, V>), dim3((unsigned)blocks), dim3(kRouteThreads), 0, s, a)
    BY_TYPE(GO)
#undef GO
    st = launch_status("route_experts");
    if (st != NNCF_AMD_OK || blocks == 1) return st;
    hipLaunchKernelGGL(k_route_place, dim3((unsigned)blocks), dim3(kRouteThreads), 0, s, a);
    return launch_status("route_experts");
}

extern "C" int nncf_amd_route_experts_grad(const void* logits, int dtype, int64_t ldl, int64_t tokens, int64_t experts, int64_t topk,
                                           int renormalize, const float* weights, const int32_t* ids, const float* dweights, void* dlogits,
                                           void* stream) {
    using namespace wc;
    const int st = check_route("route_experts_grad", dtype, tokens, experts, topk, ldl);
    if (st != NNCF_AMD_OK) return st;
    if (tokens == 0) return NNCF_AMD_OK;
    if ((!renormalize && !logits) || !weights || !ids || !dweights || !dlogits) {
        set_error("route_experts_grad: null argument");
        return NNCF_AMD_ERR_BAD_ARG;
    }
    hipStream_t s = (hipStream_t)stream;
#define GO(DT, G, V)                                                                                                              \
    hipLaunchKernelGGL((k_route_grad<DT, G, V>), dim3((unsigned)((tokens + 256 / G - 1) / (256 / G))), dim3(256), 0, s, logits, ldl, tokens, \
                       (int)experts, (int)topk, renormalize, weights, ids, dweights, dlogits)
    BY_TYPE(GO)
#undef GO
    return launch_status("route_experts_grad");
}

extern "C" int nncf_amd_combine_experts(const void* y, int in_dtype, int64_t ldy, int64_t total_rows, const float* weights, const int32_t* rows,
                                        int64_t tokens, int64_t topk, int64_t n, void* out, int out_dtype, void* stream) {
    using namespace wc;
    if ((out_dtype != NNCF_AMD_F16 && out_dtype != NNCF_AMD_BF16) || (in_dtype != NNCF_AMD_F32 && in_dtype != out_dtype)) {
        set_error("combine_experts: fp16 or bf16, and fp32 or the same for the rows (dtypes %d, %d)", in_dtype, out_dtype);
        return NNCF_AMD_ERR_DTYPE;
    }
    if (tokens < 0 || topk < 1 || n < 0 || total_rows < 0 || ldy < n || (tokens > 0 && n > 0 && (!rows || !out || (!y && total_rows > 0)))) {
        set_error("combine_experts: bad argument (tokens=%lld topk=%lld n=%lld)", (long long)tokens, (long long)topk, (long long)n);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    if (tokens == 0 || n == 0) return NNCF_AMD_OK;
    const bool wide = n % 8 == 0 && ldy % 8 == 0 && (((uintptr_t)y | (uintptr_t)out) & 15) == 0;
    const int64_t cols = wide ? n / 8 : n;
    unsigned bx = 256;
    while (bx > 8 && (int64_t)bx / 2 >= cols) bx /= 2;
    const unsigned by = 256 / bx;
    const int64_t gx = (cols + bx - 1) / bx, gy = (tokens + by - 1) / by;
    hipStream_t s = (hipStream_t)stream;
    for (int64_t y0 = 0; y0 < gy; y0 += 65535) {  // the grid's second axis ends at 65535
        const int64_t t0 = y0 * by, part = (gy - y0 < 65535 ? gy - y0 : 65535);
        const int64_t here = tokens - t0 < part * by ? tokens - t0 : part * by;
        const dim3 grid((unsigned)gx, (unsigned)part), block(bx, by);
        const float* w = weights ? weights + t0 * topk : nullptr;
        const int32_t* r = rows + t0 * topk;
        uint16_t* o = (uint16_t*)out + t0 * n;
#define GO(IN, OUT)                                                                                                          \
    if (wide) hipLaunchKernelGGL((k_combine<IN, OUT, 8>), grid, block, 0, s, y, ldy, total_rows, w, r, here, (int)topk, n, o); \
    else hipLaunchKernelGGL((k_combine<IN, OUT, 1>), grid, block, 0, s, y, ldy, total_rows, w, r, here, (int)topk, n, o)
        if (out_dtype == NNCF_AMD_BF16) {
            if (in_dtype == NNCF_AMD_F32) { GO(NNCF_AMD_F32, NNCF_AMD_BF16); }
            else { GO(NNCF_AMD_BF16, NNCF_AMD_BF16); }
        } else {
            if (in_dtype == NNCF_AMD_F32) { GO(NNCF_AMD_F32, NNCF_AMD_F16); }
            else { GO(NNCF_AMD_F16, NNCF_AMD_F16); }
        }
#undef GO
    }
    return launch_status("combine_experts");
}

extern "C" int nncf_amd_combine_experts_grad(const void* dout, int dtype, const void* y, int64_t ldy, const float* weights, const int32_t* rows,
                                             const int32_t* slots, int64_t tokens, int64_t topk, int64_t n, void* dy, float* dweights,
                                             void* stream) {
    using namespace wc;
    if (dtype != NNCF_AMD_F16 && dtype != NNCF_AMD_BF16) {
        set_error("combine_experts_grad: fp16 or bf16 (dtype %d)", dtype);
        return NNCF_AMD_ERR_DTYPE;
    }
    if (tokens < 0 || topk < 1 || n < 1 || ldy < n || tokens * topk > 0x7fffffff ||
        (tokens > 0 && (!dout || !weights || !rows || !slots || (dweights && !y)))) {
        set_error("combine_experts_grad: bad argument (tokens=%lld topk=%lld n=%lld)", (long long)tokens, (long long)topk, (long long)n);
        return NNCF_AMD_ERR_BAD_ARG;
    }
    const int64_t total = tokens * topk;
    if (total == 0 || (!dy && !dweights)) return NNCF_AMD_OK;
    const bool wide = n % 8 == 0 && ldy % 8 == 0 && (((uintptr_t)y | (uintptr_t)dout | (uintptr_t)dy) & 15) == 0;
    const dim3 grid((unsigned)((total + 3) / 4));
    hipStream_t s = (hipStream_t)stream;
#define GO(DT, VEC)                                                                                                                  \
    hipLaunchKernelGGL((k_combine_grad<DT, VEC>), grid, dim3(256), 0, s, (const uint16_t*)dout, (const uint16_t*)y, ldy, weights, rows, slots, \
                       total, (int)topk, n, (uint16_t*)dy, dweights)
    if (dtype == NNCF_AMD_BF16) {
        if (wide) GO(NNCF_AMD_BF16, 8);
        else GO(NNCF_AMD_BF16, 1);
    } else {
        if (wide) GO(NNCF_AMD_F16, 8);
        else GO(NNCF_AMD_F16, 1);
    }
#undef GO
    return launch_status("combine_experts_grad");
}
