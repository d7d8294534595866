// moe.hip - a mixture-of-experts layer on gfx950: the router, and the experts'
// products of a few tokens with what lies between them.
//
// Router (moe_route):  z = R x, scores = softmax(z) or sigmoid(z), the best
// experts by z (or by score + bias) with their scores as weights.
//
// Experts (moe_ffn), for every token t and place s with expert e = ids[t][s] >= 0:
//   g = G_e a_t,  u = U_e a_t            a_t: the token's Q8_K / Q8_0 blocks
//   h = g / (1 + exp(-g)) * u            rounded to f32, then to blocks again
//   y_t = residual_t + sum_s w_ts D_e h
// The products are those of MUL_MAT_ID (crates/tensor/src/cpu_index.rs:169-236):
// exact integers per block of 256 (or 32 for Q8_0), but added up in f64 and
// rounded once, to g, u and y.  The order of a sum's terms depends on how many
// tokens share a call (K splits, parts of a tile, and the weights of an expert that a
// token names twice).  Two orders of n terms t differ by at most 2 n 2^-53 sum|t|, so
// they round to different f32 only where a border lies in between: at most
// n 2^-28 sum|t| / |sum| of the values, e.g. one g in some millions of 4096 values
// (n = 16).  Only such a value, and an h of it that lies between two levels, can tell a
// token's company.
#include "rlq_device.hpp"
#include "rlq_igops.hpp"
#include "rlq_internal.hpp"
#include "rlq_layout.hpp"
#include "rlq_q8k.hpp"

namespace rlq {

typedef double f64x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// Router
// ---------------------------------------------------------------------------

// Four values of a row from element e on; past the end: 0.
template <bool VEC>
__device__ __forceinline__ float4 route_load(const float* p, uint32_t e, uint32_t n) {
    if constexpr (VEC) return e < n ? *(const float4*)(p + e) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    return make_float4(e < n ? p[e] : 0.0f, e + 1 < n ? p[e + 1] : 0.0f, e + 2 < n ? p[e + 2] : 0.0f,
                       e + 3 < n ? p[e + 3] : 0.0f);
}

// The maximum over the wave, in every lane (call it with every lane active).
__device__ __forceinline__ double wave_max_f64(double v) {
    auto up = [](double a, double b) { return b > a ? b : a; };
    v = up(v, dpp_d<kQuadXor1>(v));
    v = up(v, dpp_d<kQuadXor2>(v));
    v = up(v, dpp_d<kRowHalfMirror>(v));
    v = up(v, dpp_d<kRowRor8>(v));
    return up(up(readlane_d(v, 0), readlane_d(v, 16)), up(readlane_d(v, 32), readlane_d(v, 48)));
}

// The best experts of token t by one wave; lane l holds experts l, l + 64, ...
// (NI of them).  Ranks are f64 (score + bias), or with no bias the f32 logits as
// ordered u32 keys (1 and up; equal floats have equal keys): a round of the
// search is then about 30 instructions instead of 100.
// z: the token's logits in LDS, or null: in a.logits, where other workgroups may
// have put some (read at the level at which route_put's exchanges are performed).
template <int NI>
__device__ __forceinline__ void route_choose(const RouteArgs& a, uint32_t t, const float* z) {
    const uint32_t lane = threadIdx.x & 63, E = a.experts;
    float v[NI];
    int bad = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const uint32_t e = lane + 64 * i;
        v[i] = 0.0f;
        if (e < E)
            v[i] = z ? z[e] : __hip_atomic_load(a.logits + (uint64_t)t * E + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        bad |= !finite(v[i]);
    }
    int32_t* ids = a.ids + (uint64_t)t * a.slots;
    float* weights = a.weights + (uint64_t)t * a.slots;
    if (__ballot(bad)) {
        if (lane < a.slots) ids[lane] = -1, weights[lane] = 0.0f;
        if (lane == 0) report_error(a.err_word, model_key(t, kStOOut, 0));
        return;
    }
    uint32_t key[NI], best = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
        const uint32_t b = __float_as_uint(v[i] == 0.0f ? 0.0f : v[i]);
        key[i] = lane + 64 * i < E ? ((b >> 31) ? ~b : b | 0x80000000u) : 0;
        best = key[i] > best ? key[i] : best;
    }
    best = wave_max_u32(best);
    double score[NI];
    if (a.sigmoid) {
#pragma unroll
        for (int i = 0; i < NI; ++i) score[i] = 1.0 / (1.0 + exp(-(double)v[i]));
    } else {
        const double top = (double)__uint_as_float((best >> 31) ? best ^ 0x80000000u : ~best);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            score[i] = exp((double)v[i] - top);
            if (lane + 64 * i < E) sum += score[i];
        }
        sum = wave_sum_f64(sum);
#pragma unroll
        for (int i = 0; i < NI; ++i) score[i] = score[i] / sum;
    }
    int32_t id = -1;  // of place `lane`
    double weight = 0.0;
    // the lowest of the experts that `mine` marks takes place s; taken(i): it leaves
    auto take = [&](uint32_t s, auto&& mine, auto&& taken) {
        bool found = false;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            if (found) continue;  // (uniform)
            const unsigned long long m = __ballot(mine(i));
            if (!m) continue;
            found = true;
            const int l = __builtin_ctzll(m);
            const double w = readlane_d(score[i], l);
            if ((int)lane == l) taken(i);
            if (lane == s) id = l + 64 * i, weight = w;
        }
    };
    if (!a.bias) {
        for (uint32_t s = 0; s < a.slots; ++s) {  // (slots <= experts)
            take(s, [&](int i) { return key[i] == best; }, [&](int i) { key[i] = 0; });
            best = key[0];
#pragma unroll
            for (int i = 1; i < NI; ++i) best = key[i] > best ? key[i] : best;
            best = wave_max_u32(best);
        }
    } else {
        double rank[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const uint32_t e = lane + 64 * i;
            rank[i] = e < E ? score[i] + (double)a.bias[e] : -INFINITY;
            if (!(rank[i] > -INFINITY)) rank[i] = -INFINITY;  // (a bias of NaN: never chosen)
        }
        for (uint32_t s = 0; s < a.slots; ++s) {
            double most = rank[0];
#pragma unroll
            for (int i = 1; i < NI; ++i) most = rank[i] > most ? rank[i] : most;
            most = wave_max_f64(most);
            if (!(most > -INFINITY)) break;  // no expert left for the places from s on
            take(s, [&](int i) { return rank[i] == most; }, [&](int i) { rank[i] = -INFINITY; });
        }
    }
    bool none = id < 0;  // 0 times a scale that is not finite would be NaN
    if (a.normalize) {
        const double all = wave_sum_f64(weight);
        none |= !(all > 0.0);
        weight = weight / all;
    }
    if (lane < a.slots) ids[lane] = id, weights[lane] = none ? 0.0f : (float)(weight * (double)a.scale);
}

// A workgroup's logits zs[n tokens][m experts] of tokens from t0 and experts from e0
// on; then the last of the `parts` workgroups of these tokens to arrive chooses
// their experts.  With one part they are in LDS already.  Otherwise they are put
// where every workgroup can read them: an exchange is performed at the device's
// coherent level when it returns, and its result is waited for, so the count after
// the barrier needs no release (which would write the whole L2 back).
template <int W, int NI>
__device__ __forceinline__ void route_finish(const RouteArgs& a, const float* zs, uint32_t t0, uint32_t n, uint32_t e0,
                                             uint32_t m, uint32_t group, uint32_t parts) {
    __shared__ uint32_t last;
    n = a.tokens - t0 < n ? a.tokens - t0 : n;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n * m; i += 64 * W) {
        const uint32_t b = i / m, e = e0 + i - b * m;
        float* to = a.logits + (uint64_t)(t0 + b) * a.experts + e;
        if (parts == 1) {
            *to = zs[i];
        } else {
            const uint32_t old = __hip_atomic_exchange((uint32_t*)to, __float_as_uint(zs[i]), __ATOMIC_RELAXED,
                                                       __HIP_MEMORY_SCOPE_AGENT);
            asm volatile("" ::"v"(old) : "memory");
        }
    }
    if (parts > 1) {
        __syncthreads();
        if (threadIdx.x == 0) {
            const uint32_t old = __hip_atomic_fetch_add(a.count + group, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last = old == parts - 1;
            if (last) __hip_atomic_store(a.count + group, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last) return;
    }
    for (uint32_t k = threadIdx.x >> 6; k < n; k += W) route_choose<NI>(a, t0 + k, parts == 1 ? zs + k * m : nullptr);
}

// TB tokens, whose rows lie in LDS, and a run of experts per workgroup; a wave takes
// one expert at a time, 2048 values of its row in flight while the next are
// loaded, K over its lanes.
//
// Bound: a launch, two memory latencies and the choice; where workgroups have
// several experts a wave, the loads' latency (two experts at a time did not pay:
// 128 experts of 2048 values, 128 tokens 16.0 us with one, 15.7 with two; 8 of
// 4096, 512 tokens 8.4 and 12.1).  One token: 8 experts of 4096 values 4.9 us (29 as
// two launches, the products on MFMA), 128 of 2048 6.4.
template <int TB, int NI, bool VEC>
__global__ __launch_bounds__(512) void route_few_kernel(RouteArgs a) {
    extern __shared__ __align__(16) float xs[];  // [TB][K up to a multiple of 2048], logits [TB][experts of the run]
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = a.cols, E = a.experts;
    const uint32_t t0 = blockIdx.y * TB, per = (E + gridDim.x - 1) / gridDim.x, e0 = blockIdx.x * per;
    const uint32_t e1 = e0 + per < E ? e0 + per : E, pad = (K + 2047) / 2048 * 2048;
    float* zs = xs + TB * pad;
    float4 r[8];
    auto load = [&](uint32_t e, uint32_t k0) {
#pragma unroll
        for (int u = 0; u < 8; ++u) r[u] = route_load<VEC>(a.router + (uint64_t)e * K, k0 + 256 * u + 4 * lane, K);
    };
    uint32_t e = e0 + wave;
    if (e < e1) load(e, 0);
#pragma unroll
    for (int b = 0; b < TB; ++b) {
        const float* x = a.x + (uint64_t)(t0 + b < a.tokens ? t0 + b : a.tokens - 1) * K;
        for (uint32_t k = 4 * threadIdx.x; k < pad; k += 2048) *(float4*)(xs + b * pad + k) = route_load<VEC>(x, k, K);
    }
    __syncthreads();
    for (; e < e1; e += 8) {
        double z[TB][2] = {};
        for (uint32_t k0 = 0; k0 < K; k0 += 2048) {
            float4 w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) w[u] = r[u];
            if (k0 + 2048 < K) load(e, k0 + 2048);
            else if (e + 8 < e1) load(e + 8, 0);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const double rd[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
#pragma unroll
                for (int b = 0; b < TB; ++b) {
                    const float4 x = *(const float4*)(xs + b * pad + k0 + 256 * u + 4 * lane);
                    z[b][0] = __builtin_fma((double)x.x, rd[0], z[b][0]);
                    z[b][1] = __builtin_fma((double)x.y, rd[1], z[b][1]);
                    z[b][0] = __builtin_fma((double)x.z, rd[2], z[b][0]);
                    z[b][1] = __builtin_fma((double)x.w, rd[3], z[b][1]);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < TB; ++b) {
            const double v = wave_sum_f64(z[b][0] + z[b][1]);
            if (lane == 0) zs[b * (e1 - e0) + e - e0] = (float)v;
        }
    }
    route_finish<8, NI>(a, zs, t0, TB, e0, e1 - e0, blockIdx.y, gridDim.x);
}

// z of 16 tokens x 16 experts per workgroup on v_mfma_f64_16x16x4_f64, K split over
// W waves in slices of 32 (lane l holds row l % 16, values 8 (l / 16) .. + 7 of
// the slice), two slices loaded ahead, the waves' sums added in wave order.
//
// Bound: 512 tokens, 128 experts of 2048 values 19 us, of which the f64 products
// are 3.4 at the rate of the matrix cores; a launch, the sums' way through LDS, the
// exchange of the logits and the choice take 10 (measured with K = 32).
template <int W, int NI, bool VEC>
__global__ __launch_bounds__(64 * W) void route_many_kernel(RouteArgs a) {
    __shared__ double part[W][4][64];
    __shared__ float zs[256];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, kq = lane >> 4;
    const uint32_t t0 = blockIdx.y * 16, e0 = blockIdx.x * 16, m = a.experts - e0 < 16 ? a.experts - e0 : 16, K = a.cols;
    const float* x = a.x + (uint64_t)(t0 + i < a.tokens ? t0 + i : a.tokens - 1) * K;
    const float* r = a.router + (uint64_t)(e0 + i < a.experts ? e0 + i : a.experts - 1) * K;
    f64x4 acc[2] = {{0.0, 0.0, 0.0, 0.0}, {0.0, 0.0, 0.0, 0.0}};
    float4 v[2][4];
    auto load = [&](float4 (&d)[4], uint32_t k) {
        const uint32_t e = k + 8 * kq;
        d[0] = route_load<VEC>(x, e, K), d[1] = route_load<VEC>(x, e + 4, K);
        d[2] = route_load<VEC>(r, e, K), d[3] = route_load<VEC>(r, e + 4, K);
    };
    load(v[0], wave * 32);
    load(v[1], wave * 32 + W * 32);
    for (uint32_t k = wave * 32; k < K; k += 2 * W * 32) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float4(&d)[4] = v[h];
            const float xv[8] = {d[0].x, d[0].y, d[0].z, d[0].w, d[1].x, d[1].y, d[1].z, d[1].w};
            const float rv[8] = {d[2].x, d[2].y, d[2].z, d[2].w, d[3].x, d[3].y, d[3].z, d[3].w};
            load(v[h], k + (2 + h) * W * 32);
#pragma unroll
            for (int j = 0; j < 8; ++j)  // (a slice past the end is zeros)
                acc[j & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)xv[j], (double)rv[j], acc[j & 1], 0, 0, 0);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) part[wave][q][lane] = acc[0][q] + acc[1][q];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < 256; o += 64 * W) {
        // value q of lane l: token 4 q + l / 16, expert l % 16
        const uint32_t q = o >> 6, l = o & 63, e = l & 15;
        double z = 0.0;
#pragma unroll
        for (int w = 0; w < W; ++w) z += part[w][q][l];
        if (e < m) zs[(4 * q + (l >> 4)) * m + e] = (float)z;
    }
    route_finish<W, NI>(a, zs, t0, 16, e0, m, blockIdx.y, gridDim.x);
}

// The grid of route_few_kernel: a part for every eight experts (one a wave) while
// there are CUs for them, `per` experts each.
static uint32_t route_per(const RouteArgs& a, uint32_t groups) {
    const uint32_t cus = (uint32_t)device_cus(), most = cus > groups ? cus / groups : 1, eights = (a.experts + 7) / 8;
    const uint32_t parts = eights < most ? eights : most;
    return (a.experts + parts - 1) / parts;
}

template <int TB, int NI, bool VEC>
static hipError_t route_few_launch(const RouteArgs& a, uint32_t groups, uint32_t per, hipStream_t s) {
    static LdsLimit lim;
    const uint32_t lds = TB * ((a.cols + 2047) / 2048 * 2048 + per) * 4;
    const hipError_t e = lim.raise((const void*)route_few_kernel<TB, NI, VEC>, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((route_few_kernel<TB, NI, VEC>), dim3((a.experts + per - 1) / per, groups), dim3(512), lds, s, a);
    return hipGetLastError();
}

// One token a workgroup while every eight experts of every token can have a CU, else
// two (us: 64 tokens, 8 experts of 4096 values 5.7 against 6.8 with two; 128 tokens,
// 128 of 2048 16.1 against 14.0).  Such a workgroup's time grows with its steps (a
// wave's experts times 2048 values of K, times the rounds of workgroups), the MFMA
// tiles' with K alone: few / tiles, 512 tokens, 32 experts of 2048 values (4 steps)
// 11.8 / 15.4, 64 (8) 18.1 / 15.9, 128 (16) 32.0 / 19.0; 200 tokens, 60 of 896 (4) 11.6
// / 10.3; 100 tokens, 256 of 4096 (14) 26.8 / 24.8; 30 tokens, 256 of 7168 (8) 20.0 /
// 34.5.  Rows of more than 16384 values do not fit LDS.
template <int NI, bool VEC>
static hipError_t route_launch(const RouteArgs& a, hipStream_t s) {
    const uint32_t cus = (uint32_t)device_cus();
    const bool one = (uint64_t)a.tokens * ((a.experts + 7) / 8) <= cus;
    const uint32_t groups = one ? a.tokens : (a.tokens + 1) / 2, per = route_per(a, groups);
    const uint64_t rounds = ((uint64_t)groups * ((a.experts + per - 1) / per) + cus - 1) / cus;
    const uint64_t steps = (uint64_t)((per + 7) / 8) * ((a.cols + 2047) / 2048) * rounds;
    if (a.cols <= 16384 && (one || steps <= 2 + a.cols / 512))
        return one ? route_few_launch<1, NI, VEC>(a, groups, per, s) : route_few_launch<2, NI, VEC>(a, groups, per, s);
    hipLaunchKernelGGL((route_many_kernel<16, NI, VEC>), dim3((a.experts + 15) / 16, (a.tokens + 15) / 16), dim3(1024), 0, s,
                       a);
    return hipGetLastError();
}

hipError_t launch_moe_route(const RouteArgs& a, hipStream_t s) {
    if (a.tokens == 0 || a.experts == 0 || a.cols == 0 || a.experts > kMoeMaxExperts || a.slots == 0 ||
        a.slots > kMoeMaxSlots || a.slots > a.experts || a.tokens > 65535)
        return hipErrorInvalidValue;
    const bool vec = (((uintptr_t)a.x | (uintptr_t)a.router) & 15) == 0 && a.cols % 4 == 0;
    if (a.experts <= 64) return vec ? route_launch<1, true>(a, s) : route_launch<1, false>(a, s);
    if (a.experts <= 256) return vec ? route_launch<4, true>(a, s) : route_launch<4, false>(a, s);
    return vec ? route_launch<16, true>(a, s) : route_launch<16, false>(a, s);
}

// ---------------------------------------------------------------------------
// Experts: the plan and the activation images
//
// A pass takes up to 32 tokens.  Its plan lists the experts in use in ascending
// order as (expert, base, mask): the expert serves the tokens of mask, ascending, whose h
// rows start at base.  Entries past the last one have no tokens.  A token that names an expert twice
// is one column of it, with the sum of both weights.  A single token has no
// plan: its places that name an expert are read from ids where they are needed.
//
// The images hold activations in chunks of 256 values (of a Q8_0 row's last chunk, a
// part; the rest is 0), in the slot order of rlq_layout.hpp for Q4_K and Q5_K: 256
// levels, their 16 f16 sums (weights with mins) and a f64 scale (Q8_0: 8), of h times
// the token's weight for the expert.
//   x  [chunk][token], a chunk's levels in two lines of its own: an expert takes some
//      of the tokens (32 tokens, 8 experts of 14336x4096 121 us against 135 with the
//      tokens' 16-byte pieces side by side)
//   h  expert after expert, so that the down product runs over all of them as over
//      one long row; of each [chunk], and of that the pieces of its own tokens side by
//      side: q [k-step 8][k half 2][column][16 int8], sums [k half 2][column][8 f16],
//      f [column] or [k-step][column]
// A single token's images lie in LDS.
//
// A block with a data error has kMoeBad as its scale.  That NaN reaches every sum of
// its token, and who finds a sum to be a NaN looks whether the mark is among the
// scales (one with a NaN weight is no error): such a token's h is NaN, and its y is
// not written.  No other value has these bits: they are no f32's, and the result of no
// operation.
// ---------------------------------------------------------------------------
constexpr unsigned long long kMoeBad = 0x7ff8000000000001ull;
__device__ __forceinline__ double moe_bad_scale() { return __longlong_as_double((long long)kMoeBad); }
__device__ __forceinline__ bool moe_is_bad(double f) { return (unsigned long long)__double_as_longlong(f) == kMoeBad; }
// The scale of a column that a chunk does not concern, where products with it are left
// out: no scale is -0.
__device__ __forceinline__ bool moe_is_out(double f) { return (unsigned long long)__double_as_longlong(f) == 1ull << 63; }

// The places of a single token that name an expert (bit s), and whether one is out
// of range; every wave for itself.
struct MoePlaces {
    unsigned long long some;
    int32_t id;  // of place `lane`
    int wrong;   // the first place out of range, or -1
};
__device__ __forceinline__ MoePlaces moe_places(const MoeArgs& a) {
    const uint32_t lane = threadIdx.x & 63;
    MoePlaces p;
    p.id = lane < a.slots ? a.ids[lane] : -1;
    p.some = __ballot(p.id >= 0 && p.id < (int32_t)a.experts);
    const unsigned long long off = __ballot(p.id < -1 || p.id >= (int32_t)a.experts);
    p.wrong = off ? __builtin_ctzll(off) : -1;
    return p;
}

__device__ __forceinline__ void moe_plan(const MoeArgs& a) {
    __shared__ uint32_t mask[kMoeMaxExperts], wave_n[8], wave_b[8], bad, served;
    __shared__ uint16_t place[kMoeMaxExperts];
    __shared__ int32_t ids[kMoeTokens * kMoeMaxSlots];
    __shared__ float weights[kMoeTokens * kMoeMaxSlots];
    const uint32_t tid = threadIdx.x, nt = blockDim.x, lane = tid & 63, wave = tid >> 6, waves = nt >> 6;
    const uint32_t pairs = a.tokens * a.slots;
    for (uint32_t e = tid; e < a.experts; e += nt) mask[e] = 0;
    if (tid == 0) bad = 0, served = 0;
    __syncthreads();
    for (uint32_t p = tid; p < pairs; p += nt) {
        int32_t id = a.ids[p];
        const uint32_t t = p / a.slots;
        if (id >= 0 && id < (int32_t)a.experts) {
            atomicOr(&mask[id], 1u << t);
        } else if (id != -1) {
            report_error(a.err_word, bounds_key((uint64_t)a.token0 * a.slots + p));
            atomicOr(&bad, 1u << t);
            id = -1;
        }
        ids[p] = id, weights[p] = a.weights[p];
    }
    __syncthreads();
    uint32_t used = 0, rows = 0;
    for (uint32_t e0 = 0; e0 < a.experts; e0 += nt) {
        const uint32_t e = e0 + tid, m = e < a.experts ? mask[e] : 0, c = (uint32_t)__builtin_popcount(m);
        // this expert's place among the used ones, and its first row
        const unsigned long long some = __ballot(m != 0);
        uint32_t before = c;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)before, d, 64);
            if (lane >= (uint32_t)d) before += o;
        }
        if (lane == 63) wave_n[wave] = (uint32_t)__builtin_popcountll(some), wave_b[wave] = before;
        __syncthreads();
        uint32_t j = used + (uint32_t)__builtin_popcountll(some & ((1ull << lane) - 1)), b = rows + before - c;
        for (uint32_t w = 0; w < waves; ++w) {
            if (w < wave) j += wave_n[w], b += wave_b[w];
            used += wave_n[w], rows += wave_b[w];
        }
        if (m) a.plan[j] = make_uint4(e, b, m, 0), place[e] = (uint16_t)j, atomicOr(&served, m);
        __syncthreads();
    }
    for (uint32_t j = used + tid; j < a.most; j += nt) a.plan[j] = make_uint4(0, 0, 0, 0);
    if (tid == 0) *a.head = make_uint4(used, bad, served, 0);
    for (uint32_t p = tid; p < pairs; p += nt) {  // a token's first place with an expert speaks for all of them
        const int32_t id = ids[p];
        const uint32_t t = p / a.slots, end = (t + 1) * a.slots;
        bool first = id >= 0;
        for (uint32_t o = t * a.slots; o < p; ++o) first = first && ids[o] != id;
        if (!first) continue;
        double w = 0.0;
        for (uint32_t o = p; o < end; ++o)
            if (ids[o] == id) w += (double)weights[o];
        a.wsum[place[id] * kMoeTokens + t] = w;
    }
}

__device__ __forceinline__ void moe_load16(const float* p, float (&v)[16]) {
    const float4* src = (const float4*)p;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float4 w = src[k];
        v[4 * k] = w.x, v[4 * k + 1] = w.y, v[4 * k + 2] = w.z, v[4 * k + 3] = w.w;
    }
}

// One lane's 16 values (r16 of a chunk's 16 lanes) into an image for weights of type T:
// column c of n that lie side by side, the first at place `at` of the image.
template <uint32_t T>
__device__ __forceinline__ void image_put(const MoeImage& im, uint64_t at, uint32_t c, uint32_t n, uint32_t r16,
                                          const uint32_t (&q)[4], int32_t bsum, double f) {
    const uint4 w = ig_slots(T) ? q45_slots(q, r16 & 1) : make_uint4(q[0], q[1], q[2], q[3]);
    *(uint4*)(im.q + at * 256 + (r16 * n + c) * 16) = w;
    if constexpr (ig_mins(T)) im.sums[at * 16 + ((r16 >> 3) * n + c) * 8 + (r16 & 7)] = (_Float16)bsum;
    if constexpr (T == kQ8_0) {
        if (!(r16 & 1)) im.f[at * 8 + (r16 >> 1) * n + c] = f;
    } else {
        if (r16 == 0) im.f[at + c] = f;
    }
}

// Quantizes one lane's 16 values for weights of type T; returns the kind of the
// block's data error, or -1.
template <uint32_t T>
__device__ __forceinline__ int image_quantize(const float (&v)[16], uint32_t r16, uint32_t (&q)[4], float& d, int32_t& bsum,
                                              uint32_t& index) {
    if constexpr (T == kQ8_0) {
        bsum = 0;
        return q8_0_pair16(v, r16 & 1, q, d, index);
    } else {
        const Q8KRow o = q8k_row16(v, r16);
#pragma unroll
        for (int k = 0; k < 4; ++k) q[k] = o.q[k];
        d = o.d, bsum = o.bsum, index = o.index;
        return o.kind;
    }
}

// One lane's 16 values of chunk c of token t of x, from f32 rows or from packed
// blocks (taken as given; the 16-value sums are those of the levels).  report: this
// workgroup tells of a data error.
template <uint32_t T, bool PACKED>
__device__ __forceinline__ bool moe_x(const MoeArgs& a, uint32_t c, uint32_t r16, uint32_t t, bool report, uint32_t (&q)[4],
                                      int32_t& bsum, double& f) {
    const uint32_t K = a.cols, e0 = c * 256 + r16 * 16;
    float d = 0.0f;
    int kind = -1;
    bsum = 0;
    q[0] = q[1] = q[2] = q[3] = 0;
    if constexpr (PACKED) {
        if (e0 < K) {
            if constexpr (T == kQ8_0) {
                const uint16_t* b = (const uint16_t*)((const uint8_t*)a.x + ((uint64_t)t * (K / 32) + e0 / 32) * 34);
                d = half_bits_to_float_exact(b[0]);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    q[k] = (uint32_t)b[1 + 8 * (r16 & 1) + 2 * k] | (uint32_t)b[2 + 8 * (r16 & 1) + 2 * k] << 16;
            } else {
                const uint32_t* b = (const uint32_t*)((const uint8_t*)a.x + ((uint64_t)t * (K / 256) + c) * 292);
                d = __uint_as_float(b[0]);
#pragma unroll
                for (int k = 0; k < 4; ++k) q[k] = b[1 + 4 * r16 + k];
#pragma unroll
                for (int k = 0; k < 4; ++k) bsum = dot4(q[k], 0x01010101u, bsum);
            }
        }
    } else {
        float v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = 0.0f;
        if (e0 < K) moe_load16((const float*)a.x + (uint64_t)t * K + e0, v);
        uint32_t index;
        kind = image_quantize<T>(v, r16, q, d, bsum, index);
        if (kind >= 0 && report && (T == kQ8_0 ? !(r16 & 1) : r16 == 0)) {
            const uint64_t block = T == kQ8_0 ? e0 / 32 : c, first = T == kQ8_0 ? e0 / 32 * 32ull : c * 256ull;
            report_error(a.err_word, kind == kKindNonFinite ? error_key(a.token0 + t, kKindNonFinite, first + index)
                                                            : error_key(a.token0 + t, kKindScale, block));
        }
    }
    f = kind >= 0 ? moe_bad_scale() : (double)d;
    return kind >= 0;
}

// Workgroup 0: the plan.  The others: one chunk of x each, 16 lanes per token.
template <uint32_t T, bool PACKED>
__global__ __launch_bounds__(512) void moe_prepare_kernel(MoeArgs a) {
    if (blockIdx.x == 0) {
        moe_plan(a);
        return;
    }
    const uint32_t c = blockIdx.x - 1, r16 = threadIdx.x & 15, t = threadIdx.x >> 4;
    if (t >= a.tokens) return;
    bool some = false;  // x of a token without experts is not looked at
    for (uint32_t s = r16; s < a.slots; s += 16) {
        const int32_t id = a.ids[t * a.slots + s];
        some |= id >= 0 && id < (int32_t)a.experts;
    }
    some = (__ballot(some) >> (threadIdx.x & 48)) & 0xffffu;
    uint32_t q[4];
    int32_t bsum;
    double f;
    moe_x<T, PACKED>(a, c, r16, t, some, q, bsum, f);
    image_put<T>(a.xi, (uint64_t)c * a.tokens + t, 0, 1, r16, q, bsum, f);
}

// h of expert j's tokens, one chunk, into the image for down matrices of type T.  (A
// launch of its own: the workgroup of moe_up_kernel that writes the last rows of a
// chunk could do it, but the exchanges and counts by which it knows cost all of them
// more than the launch: 32 tokens, 8 experts of 14336x4096 162 us against 133 + 5.5; 5
// tokens, 16 Q8_0 experts of 1952x928 18.8 against 12.6 + 4.  In the LDS of the down
// product's workgroups, as a single token's, it takes a call of 5 tokens from 29.2 to 28.2 us, of 11,
// 32 experts of 1024x2048, from 32.9 to 33.2: not worth another form of that kernel.)
template <uint32_t T>
__global__ __launch_bounds__(512) void moe_h_kernel(MoeArgs a) {
    const uint32_t c = blockIdx.x, j = blockIdx.y, r16 = threadIdx.x & 15, t = threadIdx.x >> 4;
    const uint4 p = a.plan[j];
    if (!((p.z >> t) & 1u)) return;
    const uint32_t n = (uint32_t)__builtin_popcount(p.z), col = (uint32_t)__builtin_popcount(p.z & ((1u << t) - 1));
    const uint32_t e0 = c * 256 + r16 * 16;
    float v[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) v[k] = 0.0f;
    if (e0 < a.ffn) moe_load16(a.h + (uint64_t)(p.y + col) * a.ffn + e0, v);
    uint32_t q[4], index;
    float d;
    int32_t bsum;
    const int kind = image_quantize<T>(v, r16, q, d, bsum, index);
    if (kind == kKindScale && (T == kQ8_0 ? !(r16 & 1) : r16 == 0))  // (a non-finite h has been reported)
        report_error(a.err_word, model_key(a.token0 + t, kStDownQuant, T == kQ8_0 ? e0 / 32 : c));
    const double f = kind >= 0 ? moe_bad_scale() : a.wsum[j * kMoeTokens + t] * (double)d;
    image_put<T>(a.hi, (uint64_t)p.y * gridDim.x + c * n, col, n, r16, q, bsum, f);
}

// ---------------------------------------------------------------------------
// The products
//
// A wave multiplies 32 weight rows with up to 32 columns, a chunk of 256 values
// at a time: the weights and the activations come straight into registers, one
// chunk ahead (Ig<T>::refill), and the integers A (and B, Mn) of the chunk are
// folded into f64 sums.  Lane (ln, kh): row ln of the 32 as weights, column ln as
// activations, and of the products row ln, columns 8 (i / 4) + 4 kh + i % 4.
// The two 16-row halves hf = ln / 16 of the 32 rows are
//   up    the gate and the up tile of the same 16 rows, the columns an expert's
//         tokens: the two factors of an h lie 16 lanes apart;
//   down  the same 16-row tile at two different chunks, whose activations are
//         columns 0..15 and 16..31: a row's products are those of its own half.
// ---------------------------------------------------------------------------
template <uint32_t T>
struct MoeWeights {
    static constexpr uint32_t kChunk = Ig<T>::kChunk;
    static constexpr int kFactors = 1;
    typename Ig<T>::Raw r;
};
template <>
struct MoeWeights<kQ8_0> {
    static constexpr uint32_t kChunk = 4 * kQ80Chunk;
    static constexpr int kFactors = 8;
    uint4 q[8];
    uint32_t d[4];
};

// A workgroup's LDS: its waves' f64 sums, each wave's column scales of its current
// chunk, and (one token) the image of x (up) or of its part of h (down).
template <uint32_t T>
constexpr uint32_t moe_lds(uint32_t ks, uint32_t sums) {
    return ks * (sums * 512 + MoeWeights<T>::kFactors * 256);
}
template <uint32_t T>
constexpr uint32_t moe_lds_chunk() {
    return 256 + 32 + 8 * MoeWeights<T>::kFactors;
}
extern __shared__ __align__(16) uint8_t moe_smem[];

// Where a lane's rows have their current chunk, which place of the image it is, and
// whether it counts for the lane's column.  pairs: Q8_0 block pairs of the chunk (reading
// stops there; the image is 0 beyond).  Of h, mask: the tokens whose columns are there;
// col: the lane's one.
struct MoeAt {
    const uint8_t* w;
    uint32_t chunk, pairs;
    bool live;
    uint32_t mask, col;
    __device__ uint32_t columns() const { return (uint32_t)__builtin_popcount(mask); }
};

// Activations: of one token in LDS, of x and of h in global memory (images are below 4 GiB).
template <uint32_t T>
struct MoeLds {
    static constexpr bool kStaged = true;
    uint32_t q, sums, f;  // offsets in moe_smem
    __device__ MoeLds(uint32_t at, uint32_t chunks) : q(at), sums(at + chunks * 256), f(at + chunks * 288) {}
    __device__ i32x4 act(const MoeAt& p, int s, uint32_t kh) const {
        return *(const i32x4*)(moe_smem + q + (p.chunk * 16 + s * 2 + kh) * 16);
    }
    __device__ double scale(const MoeAt& p, int k) const {
        return *(const double*)(moe_smem + f + (p.chunk * MoeWeights<T>::kFactors + k) * 8);
    }
    __device__ f16x8 sums8(const MoeAt& p, uint32_t kh) const { return *(const f16x8*)(moe_smem + sums + (p.chunk * 2 + kh) * 16); }
    __device__ void put(uint32_t c, uint32_t r16, const uint32_t (&v)[4], int32_t bsum, double sc) const {
        const uint4 w = ig_slots(T) ? q45_slots(v, r16 & 1) : make_uint4(v[0], v[1], v[2], v[3]);
        *(uint4*)(moe_smem + q + (c * 16 + r16) * 16) = w;
        if (ig_mins(T)) *(_Float16*)(moe_smem + sums + c * 32 + r16 * 2) = (_Float16)bsum;
        if (T == kQ8_0) {
            if (!(r16 & 1)) *(double*)(moe_smem + f + (c * 8 + (r16 >> 1)) * 8) = sc;
        } else {
            if (r16 == 0) *(double*)(moe_smem + f + c * 8) = sc;
        }
    }
};
template <uint32_t T>
struct MoeX {
    static constexpr bool kStaged = false;
    const MoeImage& im;
    uint32_t tokens, tok;  // tok: the lane's column
    __device__ uint32_t place(const MoeAt& p) const { return p.chunk * tokens + tok; }
    __device__ i32x4 act(const MoeAt& p, int s, uint32_t kh) const {
        return *(const i32x4*)(im.q + (uint64_t)(place(p) * 256 + kh * 16) + s * 32);
    }
    __device__ double scale(const MoeAt& p, int k) const { return im.f[(uint64_t)(place(p) * MoeWeights<T>::kFactors) + k]; }
    __device__ f16x8 sums8(const MoeAt& p, uint32_t kh) const { return *(const f16x8*)(im.sums + (place(p) * 16 + kh * 8)); }
};
template <uint32_t T>
struct MoeH {
    static constexpr bool kStaged = false;
    const MoeImage& im;
    __device__ i32x4 act(const MoeAt& p, int s, uint32_t kh) const {
        return *(const i32x4*)(im.q + (p.chunk * 16 + (s * 2 + kh) * p.columns() + p.col) * 16);
    }
    __device__ double scale(const MoeAt& p, int k) const {
        return im.f[p.chunk * MoeWeights<T>::kFactors + k * p.columns() + p.col];
    }
    __device__ f16x8 sums8(const MoeAt& p, uint32_t kh) const {
        return *(const f16x8*)(im.sums + (p.chunk * 2 + kh * p.columns() + p.col) * 8);
    }
};

// b where mask is all ones, a where it is 0.  (A plain choice between two elements of
// a product becomes one element at a variable place, which costs a compare and a
// move for each of the sixteen.)
__device__ __forceinline__ uint32_t bits_or(uint32_t mask, uint32_t a, uint32_t b) { return (mask & b) | (~mask & a); }

// One wave's chunks of src.  at(it): where step it is.  stage(): called once, by every
// wave, while the first weights are on their way.  fold(f, term): adds a chunk's
// (Q8_0: a block's) products, term(i, fa, y) being y plus fa times product i of the
// lane's row; f: the 32 column scales, 0 where the chunk is not the column's.  GUARD:
// there the products are left out, as weights may have scales that are not finite
// (the scale is then -0, which none is otherwise).  HALVES: rows of the second half take the
// columns from 16 on.  R: k-steps whose activations are in flight.
template <uint32_t T, bool HALVES, int R, bool GUARD, typename Src, typename At, typename Stage, typename Fold>
__device__ __forceinline__ void moe_walk(const Src& src, uint32_t steps, uint32_t ln, uint32_t kh, double* fd, At&& at,
                                         Stage&& stage, Fold&& fold) {
    using M = MoeWeights<T>;
    if (steps == 0) {
        stage();
        return;
    }
    const uint32_t n = ln & 15;
    const uint32_t upper = HALVES && ln >= 16 ? ~0u : 0u;
    M m;
    i32x4 act[R];
    f16x8 bs;
    double f[M::kFactors];
    auto load_act = [&](int s, const MoeAt& p) { act[s % R] = src.act(p, s, kh); };
    auto load_scales = [&](const MoeAt& p) {
#pragma unroll
        for (int k = 0; k < M::kFactors; ++k) {
            const double v = src.scale(p, k);
            f[k] = GUARD ? (p.live ? v + 0.0 : -0.0) : (p.live ? v : 0.0);
        }
        if constexpr (ig_mins(T)) bs = src.sums8(p, kh);
    };
    auto pair_of = [&](const MoeAt& p, uint32_t k) { return p.w + (k < p.pairs ? k : p.pairs - 1) * kQ80Chunk; };
    auto load_q8 = [&](const MoeAt& p, int s) {
        if constexpr (T == kQ8_0) m.q[s] = ig_ld16(pair_of(p, s / 2) + (16 * (2 * (s & 1) + kh) + n) * 16);
    };
    auto load_d8 = [&](const MoeAt& p) {
        if constexpr (T == kQ8_0) {
#pragma unroll
            for (int k = 0; k < 4; ++k) m.d[k] = *(const uint32_t*)(pair_of(p, k) + 1024 + n * 4);
        }
    };
    MoeAt p = at(0);
    auto first_acts = [&] {
#pragma unroll
        for (int s = 0; s < R; ++s) load_act(s, p);
        load_scales(p);
    };
    if (!Src::kStaged) first_acts();
    if constexpr (T == kQ8_0) {
#pragma unroll
        for (int s = 0; s < 8; ++s) load_q8(p, s);
        load_d8(p);
    } else {
        ig_load<T>(m.r, p.w, n, kh);
    }
    stage();
    if (Src::kStaged) first_acts();
    // one step; more: the next step's loads follow the last use of what they replace
    auto step = [&](auto more_, uint32_t it) {
        constexpr bool more = decltype(more_)::value;
        MoeAt nx = p;
        if (more) nx = at(it + 1);
        if (kh == 0) {
#pragma unroll
            for (int k = 0; k < M::kFactors; ++k) fd[k * 32 + ln] = f[k];
        }
        auto next_act = [&](int s) {
            if (s + R < 8) load_act(s + R, p);
            else if (more) load_act(s + R - 8, nx);
        };
        if constexpr (T == kQ8_0) {
            uint32_t dw4[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) dw4[k] = m.d[k];
            if (more) load_d8(nx), load_scales(nx);
#pragma unroll
            for (int s = 0; s < 8; ++s) {
                const i32x4 w = __builtin_bit_cast(i32x4, m.q[s]);
                const double dw = (double)half_to_float((s & 1) ? dw4[s / 2] >> 16 : dw4[s / 2]);
                const i32x16 I = ig_mfma(act[s % R], w, (i32x16){});
                if (more) load_q8(nx, s);
                next_act(s);
                fold(fd + s * 32, [&](int i, double fa, double y) {
                    if (GUARD && moe_is_out(fa)) return y;
                    const int32_t v = HALVES ? (int32_t)bits_or(upper, I[i], I[i + 8 * HALVES]) : I[i];
                    return __builtin_fma((double)v, fa * dw, y);
                });
            }
        } else {
            using W = Ig<T>;
            const typename W::Pre pre = W::pre(m.r, kh);
            const double d = (double)W::d(m.r);
            double dmin = 0.0;
            f16x8 mins = {};
            if constexpr (ig_mins(T)) dmin = (double)W::dmin(m.r), mins = W::mins(m.r, kh);
            if (more) W::head(m.r, nx.w, n);
            i32x16 A = {}, B = {};
            ig_steps([&](auto s_) {
                constexpr int S = decltype(s_)::value;
                i32x4 wa, wb;
                W::template ops<S>(m.r, pre, wa, wb);
                A = ig_mfma(act[S % R], wa, A);
                if (W::kPlanes == 2) B = ig_mfma(act[S % R], wb, B);
                if (more) W::template refill<S>(m.r, nx.w, n, kh);
                next_act(S);
            });
            f32x16 mn = {};
            if constexpr (ig_mins(T)) mn = __builtin_amdgcn_mfma_f32_32x32x16_f16(bs, mins, (f32x16){}, 0, 0, 0);
            if (more) load_scales(nx);
            fold(fd, [&](int i, double fa, double y) {
                if (GUARD && moe_is_out(fa)) return y;
                auto block = [&](int k) {
                    return W::kPlanes == 2 ? ((uint32_t)A[k] << W::kShift) + (uint32_t)B[k] : (uint32_t)A[k];
                };
                uint32_t I = block(i);
                if constexpr (HALVES) I = bits_or(upper, I, block(i + 8));
                double v = d * (double)(int32_t)I;  // exact: 11 and 31 bits
                if constexpr (ig_mins(T)) {
                    float m = mn[i];
                    if constexpr (HALVES) m = __uint_as_float(bits_or(upper, __float_as_uint(m), __float_as_uint(mn[i + 8])));
                    v = __builtin_fma(-dmin, (double)m, v);
                }
                return __builtin_fma(fa, v, y);
            });
        }
        p = nx;
    };
    for (uint32_t it = 0; it + 1 < steps; ++it) step(std::true_type{}, it);
    step(std::false_type{}, steps - 1);
}

// Q8_0 block pairs of chunk c of a row with npairs of them (other types: unused).
__device__ __forceinline__ uint32_t moe_pairs(uint32_t npairs, uint32_t c) {
    const uint32_t left = npairs - 4 * c;
    return left < 4 ? left : 4;
}

// h of 16 rows for expert j's tokens: wave kg takes every KS-th chunk of K.  NQ:
// groups of eight columns that the tokens of the pass can need.
//
// Registers decide how many chunks a CU has in flight: four waves a SIMD to eight
// columns, three beyond, whose sums would spill (8 experts of 14336x4096 Q4_K, 16
// tokens 113 us against 123 with four).  Half a chunk's activations are loaded ahead; a
// whole one gains nothing.
//
// Bound: memory, 8 tokens 5.3 TB/s of weights; from 16 tokens on the matrix cores and
// the vector units next to it (111 us, 32 tokens 128).  Small experts are over
// before the memory is busy: 4 tokens, 64 of 1536x2048 Q5_K 27 us, 3.6 TB/s.
//
// kMoeOne, kMoeOnePacked: a single token, without a plan: every workgroup reads the
// ids and makes the image of x in LDS while its first weights are on their way (8 experts
// of 14336x4096, top-2, 28 to 36 us; with a launch for the image 5 more).
enum MoeFrom { kMoePlan, kMoeOne, kMoeOnePacked };
template <uint32_t T, int KS, int NQ, MoeFrom FROM>
__global__ __launch_bounds__(64 * KS) __attribute__((amdgpu_waves_per_eu(NQ >= 2 ? 3 : 4))) void
moe_up_kernel(MoeArgs a) {
    constexpr bool ONE = FROM != kMoePlan;
    constexpr uint32_t kF = MoeWeights<T>::kFactors;
    __shared__ uint32_t bad;
    const uint32_t lane = threadIdx.x & 63, kg = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t ln = lane & 31, kh = lane >> 5;
    const uint32_t j = blockIdx.x / a.up_tiles, tile = blockIdx.x - j * a.up_tiles;
    uint32_t mask = 1, base = j, expert;
    if constexpr (ONE) {
        const MoePlaces p = moe_places(a);
        if (p.wrong >= 0) {
            if (blockIdx.x == 0 && threadIdx.x == 0) report_error(a.err_word, bounds_key((uint64_t)a.token0 * a.slots + p.wrong));
            return;
        }
        if (j >= (uint32_t)__builtin_popcountll(p.some)) return;
        unsigned long long left = p.some;
        for (uint32_t k = 0; k < j; ++k) left &= left - 1;
        expert = (uint32_t)__builtin_amdgcn_readlane(p.id, __builtin_ctzll(left));
    } else {
        const uint4 p = a.plan[j];
        if (!p.z) return;
        expert = p.x, base = p.y, mask = p.z;
        // (knowing that there is a column, the compiler drops the first branch of the folds, lets
        // the folds of Q8_0's blocks run into each other, and spills)
        asm volatile("" : "+s"(mask));
    }
    const uint32_t live = (uint32_t)__builtin_popcount(mask), nchunk = a.x_chunks;
    const uint8_t* wt = ((ln >> 4) ? a.up : a.gate) + (uint64_t)expert * a.up_bytes + (uint64_t)tile * a.x_row_bytes;
    double* part = (double*)moe_smem;
    double* fd = part + KS * NQ * 4 * 64 + kg * (kF * 32);
    double y[NQ * 4];
#pragma unroll
    for (int i = 0; i < NQ * 4; ++i) y[i] = 0.0;
    const uint32_t steps = kg < nchunk ? (nchunk - 1 - kg) / KS + 1 : 0;
    const MoeLds<T> xs(moe_lds<T>(KS, NQ * 4), nchunk);
    auto at = [&](uint32_t it) {
        const uint32_t c = kg + it * KS;
        return MoeAt{wt + (uint64_t)c * MoeWeights<T>::kChunk, c, moe_pairs(a.x_pairs, c), true, 0, 0};
    };
    auto fold = [&](const double* f, auto&& term) {
#pragma unroll
        for (int q = 0; q < NQ; ++q)
            if ((uint32_t)(8 * q) < live) {
#pragma unroll
                for (int k = 0; k < 4; ++k) y[4 * q + k] = term(4 * q + k, f[8 * q + 4 * kh + k], y[4 * q + k]);
            }
    };
    if constexpr (ONE) {
        auto stage = [&] {
            if (threadIdx.x == 0) bad = 0;
            __syncthreads();
            for (uint32_t c = threadIdx.x >> 4; c < nchunk; c += 4 * KS) {
                uint32_t q[4];
                int32_t bsum;
                double f;
                if (moe_x<T, FROM == kMoeOnePacked>(a, c, lane & 15, 0, blockIdx.x == 0, q, bsum, f)) bad = 1;
                xs.put(c, lane & 15, q, bsum, f);
            }
            __syncthreads();
        };
        moe_walk<T, false, 4, false>(xs, steps, ln, kh, fd, at, stage, fold);
    } else {
        // lane k: the token of column k (of a column past the last one the first one's)
        const bool mine = lane < kMoeTokens && (mask >> lane) & 1u;
        const int to = mine ? __builtin_popcount(mask & ((1u << lane) - 1)) : 63;
        const uint32_t tok = (uint32_t)__builtin_amdgcn_ds_permute(4 * to, (int)lane);
        const MoeX<T> x{a.xi, a.tokens, (uint32_t)__shfl((int)tok, ln < live ? (int)ln : 0, 64) & (kMoeTokens - 1)};
        moe_walk<T, false, 4, false>(x, steps, ln, kh, fd, at, [] {}, fold);
    }
#pragma unroll
    for (int i = 0; i < NQ * 4; ++i) part[(kg * NQ * 4 + i) * 64 + lane] = y[i];
    __syncthreads();
    for (uint32_t o = threadIdx.x; o < live * 16; o += 64 * KS) {
        const uint32_t c = o >> 4, r = o & 15, i = 4 * (c >> 3) + (c & 3), l = ((c >> 2) & 1) * 32 + r;
        double g = 0.0, u = 0.0;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            g += part[(k * NQ * 4 + i) * 64 + l];
            u += part[(k * NQ * 4 + i) * 64 + l + 16];
        }
        const double gf = (double)(float)g, uf = (double)(float)u;
        float h = (float)(gf / (1.0 + exp(-gf)) * uf);
        if (!finite(h)) {
            uint32_t left = mask;  // (a single token's: 1)
            for (uint32_t k = 0; k < c; ++k) left &= left - 1;
            const uint32_t t = (uint32_t)__builtin_ctz(left);
            bool marked = ONE && bad != 0;
            if constexpr (!ONE) {
                for (uint64_t k = 0; k < nchunk * kF; ++k) marked |= moe_is_bad(a.xi.f[(k / kF * a.tokens + t) * kF + k % kF]);
            }
            if (marked) h = __builtin_nanf("");
            else report_error(a.err_word, model_key(a.token0 + t, kStDownIn, 0));
        }
        a.h[(uint64_t)(base + c) * a.ffn + tile * 16 + r] = h;
    }
}

// y of a tile of rows for every token, over the h of all experts in use as one long
// row of chunks, of which the workgroup takes its part and its waves take turns.
//   up to 16 tokens  16 rows (HALVES): a pair of chunks at a time, one for each half
//   more             32 rows: a chunk at a time, all 32 columns
// Bound: memory; one token of top-2, 56 chunks each, 4096 rows of Q6_K 28 us (3.4 TB/s),
// Q4_K 19 to 22; 8 tokens, 8 experts 55 us (4.8), 16 60, 32 72.  Six experts of 6 chunks take
// 10.5: a launch, two latencies and the joining.
//
// Where the tiles alone leave CUs idle, `parts` workgroups share a tile: they put
// their f64 sums where all can read them (by exchanges whose results are waited for,
// as the router does), and the last to arrive adds them in part order.
//
// ONE: a single token.  Every workgroup reads the ids, and makes the image of its part
// of h in LDS while its first weights are on their way.
template <uint32_t T, int KS, int NQ, bool ONE>
__global__ __launch_bounds__(64 * KS) __attribute__((amdgpu_waves_per_eu(KS == 16 ? 4 : 3))) void
moe_down_kernel(MoeArgs a) {
    constexpr bool HALVES = NQ < 4;
    constexpr uint32_t kRows = HALVES ? 16 : 32, kStep = HALVES ? 2 : 1;
    __shared__ uint2 plan[ONE ? kMoeMaxSlots : kMoeMaxExperts];  // expert | base << 16, mask
    __shared__ float weight[ONE ? kMoeMaxSlots : 1];
    __shared__ uint32_t last, marked;
    const uint32_t lane = threadIdx.x & 63, kg = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t ln = lane & 31, kh = lane >> 5, hf = ln >> 4;
    const uint32_t tile = blockIdx.x / a.parts, part = blockIdx.x - tile * a.parts;
    const uint32_t nchunk = a.h_chunks;
    uint32_t used, bad = 0, some;  // bad: tokens whose ids are out of range; some: those with an expert
    if constexpr (ONE) {
        const MoePlaces p = moe_places(a);
        bad = p.wrong >= 0;
        used = bad ? 0 : (uint32_t)__builtin_popcountll(p.some);
        some = used != 0;
        if (kg == 0 && ((p.some >> lane) & 1)) {
            const uint32_t j = (uint32_t)__builtin_popcountll(p.some & ((1ull << lane) - 1));
            plan[j] = make_uint2((uint32_t)p.id, 1), weight[j] = a.weights[lane];
        }
        if (threadIdx.x == 0) marked = 0;
    } else {
        const uint4 h = *a.head;
        used = h.x, bad = h.y, some = h.z;
        for (uint32_t i = threadIdx.x; i < a.most; i += 64 * KS) {  // (past `used` no one looks)
            const uint4 p = a.plan[i];
            plan[i] = make_uint2(p.x | p.y << 16, p.z);
        }
    }
    __syncthreads();
    // this part's chunks, whole steps of them but for the last part's end
    const uint32_t all = used * nchunk, steps_all = (all + kStep - 1) / kStep;
    const uint32_t c0 = (uint32_t)((uint64_t)steps_all * part / a.parts) * kStep;
    const uint32_t c1 = part + 1 < a.parts ? (uint32_t)((uint64_t)steps_all * (part + 1) / a.parts) * kStep : all;
    const uint32_t tok = HALVES ? ln & 15 : ln;  // the lane's column
    uint32_t t16 = HALVES ? tile : 2 * tile + hf;
    t16 = t16 < a.out_tiles ? t16 : a.out_tiles - 1;  // (rows past the end are never stored)
    const uint8_t* wt = a.down + (uint64_t)t16 * a.h_row_bytes;
    constexpr int kSums = NQ * 4;
    constexpr uint32_t kF = MoeWeights<T>::kFactors;
    double* sums = (double*)moe_smem;
    double* fd = sums + KS * kSums * 64 + kg * (kF * 32);
    double y[kSums];
#pragma unroll
    for (int i = 0; i < kSums; ++i) y[i] = 0.0;
    const uint32_t first = c0 + kStep * kg, steps = first < c1 ? (c1 - 1 - first) / (kStep * KS) + 1 : 0;
    auto at = [&](uint32_t it) {
        const uint32_t want = first + it * (kStep * KS) + (HALVES ? hf : 0), i = want < c1 ? want : c1 - 1;
        const uint32_t j = i / nchunk, c = i - j * nchunk;
        const uint2 p = plan[j];
        const uint8_t* w = wt + (uint64_t)(p.x & 0xffffu) * a.down_bytes + (uint64_t)c * MoeWeights<T>::kChunk;
        const uint32_t pairs = moe_pairs(a.h_pairs, c);
        if constexpr (ONE) return MoeAt{w, i - c0, pairs, want < c1, 1, 0};
        const bool mine = (p.y >> tok) & 1u;  // others take the first column's levels, with no scale
        const uint32_t n = (uint32_t)__builtin_popcount(p.y), before = (uint32_t)__builtin_popcount(p.y & ((1u << tok) - 1));
        return MoeAt{w, (p.x >> 16) * nchunk + c * n, pairs, mine && want < c1, p.y, mine ? before : 0};
    };
    auto fold = [&](const double* f, auto&& term) {
#pragma unroll
        for (int i = 0; i < kSums; ++i) y[i] = term(i, f[(HALVES ? 16 * hf : 0) + 8 * (i / 4) + 4 * kh + i % 4], y[i]);
    };
    // A sum that is not finite: once more, with the products that are not the column's
    // left out.
    auto again = [&] {
        double all = 0.0;
#pragma unroll
        for (int i = 0; i < kSums; ++i) all += y[i] - y[i];
        if (!__ballot(all != 0.0)) return false;
#pragma unroll
        for (int i = 0; i < kSums; ++i) y[i] = 0.0;
        return true;
    };
    if constexpr (ONE) {
        const MoeLds<T> hs(moe_lds<T>(KS, kSums), c1 - c0);
        auto stage = [&] {
            const uint32_t r16 = lane & 15;
            for (uint32_t i = c0 + (threadIdx.x >> 4); i < c1; i += 4 * KS) {
                const uint32_t j = i / nchunk, c = i - j * nchunk, e0 = c * 256 + r16 * 16;
                float v[16], d;
#pragma unroll
                for (int k = 0; k < 16; ++k) v[k] = 0.0f;
                if (e0 < a.ffn) moe_load16(a.h + (uint64_t)j * a.ffn + e0, v);
                uint32_t q[4], index;
                int32_t bsum;
                const int kind = image_quantize<T>(v, r16, q, d, bsum, index);
                if (kind >= 0) marked = 1;
                if (kind == kKindScale && tile == 0 && (T == kQ8_0 ? !(r16 & 1) : r16 == 0))
                    report_error(a.err_word, model_key(a.token0, kStDownQuant, T == kQ8_0 ? e0 / 32 : c));
                hs.put(i - c0, r16, q, bsum, (double)weight[j] * (double)d);
            }
            __syncthreads();
        };
        moe_walk<T, HALVES, 2, false>(hs, steps, ln, kh, fd, at, stage, fold);
        if (again()) moe_walk<T, HALVES, 2, true>(hs, steps, ln, kh, fd, at, [] {}, fold);
    } else {
        moe_walk<T, HALVES, 4, false>(MoeH<T>{a.hi}, steps, ln, kh, fd, at, [] {}, fold);
        if (again()) moe_walk<T, HALVES, 4, true>(MoeH<T>{a.hi}, steps, ln, kh, fd, at, [] {}, fold);
    }
#pragma unroll
    for (int i = 0; i < kSums; ++i) sums[(kg * kSums + i) * 64 + lane] = y[i];
    __syncthreads();
    // value o: row o % kRows of token o / kRows
    auto total = [&](uint32_t o) {
        const uint32_t t = o / kRows, r = o % kRows, i = 4 * (t >> 3) + (t & 3), l = ((t >> 2) & 1) * 32 + r;
        double v = 0.0;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            v += sums[(k * kSums + i) * 64 + l];
            if (HALVES) v += sums[(k * kSums + i) * 64 + l + 16];
        }
        bool off = ONE && marked != 0;
        if (!ONE && v != v) {
            for (uint32_t c = c0; c < c1 && !off; ++c) {
                const uint2 p = plan[c / nchunk];
                if (!((p.y >> t) & 1u)) continue;
                const uint32_t n = (uint32_t)__builtin_popcount(p.y), at = ((p.x >> 16) * nchunk + c % nchunk * n) * kF;
                for (uint32_t k = 0; k < kF; ++k)
                    off |= moe_is_bad(a.hi.f[at + k * n + (uint32_t)__builtin_popcount(p.y & ((1u << t) - 1))]);
            }
        }
        return off ? moe_bad_scale() : v;
    };
    auto store = [&](uint32_t o, double v) {
        const uint32_t t = o / kRows, row = tile * kRows + o % kRows;
        if (row >= a.out_rows || ((bad >> t) & 1) || moe_is_bad(v)) return;
        const uint64_t to = (uint64_t)t * a.out_rows + row;
        // (without an expert the residual as it is: a sum with +0 would take -0's sign)
        a.y[to] = !a.residual ? (float)v : (some >> t) & 1 ? (float)((double)a.residual[to] + v) : a.residual[to];
    };
    const uint32_t n = a.tokens * kRows;
    if (a.parts == 1) {
        for (uint32_t o = threadIdx.x; o < n; o += 64 * KS) store(o, total(o));
        return;
    }
    unsigned long long* mine = a.sums + ((uint64_t)tile * a.parts + part) * n;
    for (uint32_t o = threadIdx.x; o < n; o += 64 * KS) {
        const unsigned long long old = __hip_atomic_exchange(mine + o, (unsigned long long)__double_as_longlong(total(o)),
                                                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::"v"(old) : "memory");
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t old = __hip_atomic_fetch_add(a.count + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = old == a.parts - 1;
        if (last) __hip_atomic_store(a.count + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!last) return;
    for (uint32_t o = threadIdx.x; o < n; o += 64 * KS) {
        double v = 0.0;
        bool off = false;
        for (uint32_t p = 0; p < a.parts; ++p) {
            const double one = __longlong_as_double((long long)__hip_atomic_load(
                a.sums + ((uint64_t)tile * a.parts + p) * n + o, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
            off |= moe_is_bad(one);
            v += one;
        }
        store(o, off ? moe_bad_scale() : v);
    }
}

// ---------------------------------------------------------------------------
// Launch
// ---------------------------------------------------------------------------
static uint64_t moe_align(uint64_t v) { return (v + 255) & ~255ull; }
static uint64_t moe_chunks(uint64_t cols) { return (cols + 255) / 256; }

// Row tiles of the down product: 16 rows to 16 tokens, then 32.
static uint64_t moe_out_tiles(const MoeCall& c, uint32_t tokens) {
    const uint64_t t = layout_tiles(c.out_rows);
    return tokens <= 16 ? t : (t + 1) / 2;
}
// Workgroups that share a tile of the down product: as many as there are CUs for, but
// a step for every wave of each (us with 1 / 2 / 4, the rule's number first: 2: 4096 rows, 32
// tokens, 8 experts of 56 chunks 106 / 73 / 84; 4: 928 rows, 5 tokens, 16 experts of 8
// chunks of Q8_0 14.1 / 11.4 / 10.8; 2: 2048 rows, 16 tokens, 64 experts of 6 chunks 54 / 34
// / 40; 1: 4096 rows, 8 tokens, 8 experts of 56 chunks 55 / 60 / 73).
static uint32_t moe_parts(const MoeCall& c, uint32_t tokens) {
    const uint64_t tiles = moe_out_tiles(c, tokens), pairs = (uint64_t)tokens * c.slots;
    const uint64_t chunks = (pairs < c.experts ? pairs : c.experts) * moe_chunks(c.ffn);
    // 16 or 12 waves that take a pair of chunks a step, or 12 that take one
    const uint64_t step = tokens <= 8 ? 32 : tokens <= 16 ? 24 : 12, steps = (chunks + step - 1) / step;
    uint64_t parts = (uint64_t)device_cus() / tiles;
    parts = parts < steps ? parts : steps;
    return (uint32_t)(parts < 1 ? 1 : parts < 8 ? parts : 8);
}
// The scratch of a pass; base null: only its size.
static size_t moe_carve(const MoeCall& c, uint32_t tokens, uint8_t* base, MoeArgs* a) {
    uint64_t at = 0;
    auto take = [&](uint64_t bytes) {
        uint8_t* p = base + at;
        at += moe_align(bytes);
        return p;
    };
    auto image = [&](uint32_t t, uint64_t places) {
        MoeImage im;
        im.q = take(places * 256);
        im.sums = (_Float16*)take(ig_mins(t) ? places * 32 : 0);
        im.f = (double*)take(places * (t == kQ8_0 ? 64 : 8));
        return im;
    };
    const uint64_t pairs = (uint64_t)tokens * c.slots;
    const uint64_t used = pairs < c.experts || tokens == 1 ? pairs : c.experts;  // (one token: its places, each on its own)
    MoeArgs m{};
    m.head = (uint4*)take(16);
    m.plan = (uint4*)take(used * 16);
    m.most = (uint32_t)used;
    m.wsum = (double*)take(used * kMoeTokens * 8);
    m.xi = image(c.up_type, moe_chunks(c.cols) * tokens);
    m.h = (float*)take(pairs * c.ffn * 4);
    m.parts = moe_parts(c, tokens);
    m.sums = (unsigned long long*)take(m.parts > 1 ? moe_out_tiles(c, tokens) * m.parts * tokens * (tokens <= 16 ? 16 : 32) * 8 : 0);
    m.hi = image(c.down_type, pairs * moe_chunks(c.ffn));
    if (a) *a = m;
    return at;
}

// What the largest of a call's passes needs (the last one may have fewer tokens).
size_t moe_bytes(const MoeCall& c) {
    const size_t most = moe_carve(c, c.tokens < kMoeTokens ? (uint32_t)c.tokens : kMoeTokens, nullptr, nullptr);
    const uint32_t rest = (uint32_t)(c.tokens % kMoeTokens);
    const size_t last = rest ? moe_carve(c, rest, nullptr, nullptr) : 0;
    return most > last ? most : last;
}

// Arrival counters: one per tile of the down product.
uint64_t moe_counters(const MoeCall& c) { return layout_tiles(c.out_rows); }

// Whether every launch of the call stays below 2^32 threads and its images of x and
// h below 4 GiB.
bool moe_takes(const MoeCall& c) {
    const uint64_t t = c.tokens < kMoeTokens ? c.tokens : kMoeTokens;
    uint64_t used = t * c.slots < c.experts ? t * c.slots : c.experts;
    used = used > c.slots ? used : c.slots;  // (a last token on its own)
    return c.experts <= kMoeMaxExperts && c.slots <= kMoeMaxSlots && c.tokens <= 65535 && c.cols <= (1u << 30) &&
           c.ffn <= (1u << 30) && used * layout_tiles(c.ffn) * 1024 <= 0xffffffffull &&
           layout_tiles(c.out_rows) * 8 * 1024 <= 0xffffffffull && used * moe_chunks(c.ffn) * 512 <= 0xffffffffull &&
           (moe_chunks(c.cols) + 1) * 512 <= 0xffffffffull && t * moe_chunks(c.cols) * 256 <= 0xffffffffull &&
           t * c.slots * moe_chunks(c.ffn) * 256 <= 0xffffffffull;
}

// Chunks of h that a workgroup of the down product has at most, of a single token.
static uint32_t moe_one_chunks(const MoeArgs& a) {
    const uint32_t all = a.slots * a.h_chunks;
    return (all + a.parts - 1) / a.parts + 2;  // (a part is whole pairs)
}
// A single token whose x and h fit LDS takes two launches, others four.
// (Q8_0's images are the largest: 256 chunks of h beside the waves' sums are 152 KB.  One
// token, 64 experts of 1536x2048 Q5_K, top-6: 21 us a call with two launches, 27 with four.)
static bool moe_one(const MoeArgs& a) { return a.tokens == 1 && a.x_chunks <= 128 && moe_one_chunks(a) <= 256; }

template <uint32_t T, int KS, int NQ, MoeFrom FROM>
static hipError_t moe_up_launch(const MoeArgs& a, uint32_t used, hipStream_t s) {
    static LdsLimit lim;
    const uint32_t lds = moe_lds<T>(KS, NQ * 4) + (FROM == kMoePlan ? 0 : a.x_chunks * moe_lds_chunk<T>());
    const hipError_t e = lim.raise((const void*)moe_up_kernel<T, KS, NQ, FROM>, lds + 64);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((moe_up_kernel<T, KS, NQ, FROM>), dim3(used * a.up_tiles), dim3(64 * KS), lds, s, a);
    return hipGetLastError();
}
template <uint32_t T, int KS, int NQ, bool ONE>
static hipError_t moe_down_launch(const MoeArgs& a, hipStream_t s) {
    static LdsLimit lim;
    constexpr uint32_t tiles = NQ < 4 ? 1 : 2;
    const uint32_t lds = moe_lds<T>(KS, NQ * 4) + (ONE ? moe_one_chunks(a) * moe_lds_chunk<T>() : 0);
    const hipError_t e = lim.raise((const void*)moe_down_kernel<T, KS, NQ, ONE>, lds + (ONE ? kMoeMaxSlots : kMoeMaxExperts) * 8 + 512);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((moe_down_kernel<T, KS, NQ, ONE>), dim3((a.out_tiles + tiles - 1) / tiles * a.parts), dim3(64 * KS),
                       lds, s, a);
    return hipGetLastError();
}

template <uint32_t T>
static hipError_t moe_up_any(const MoeArgs& a, bool packed, uint32_t used, hipStream_t s) {
    if (moe_one(a)) {
        // K over two waves where the tiles can keep the CUs busy by themselves, else over four (us with
        // 2 / 4, one token of top-2: 896 tiles an expert of 16 chunks 36.0 / 38.3, 512 of 32 34.4 /
        // 41.1; top-8, 96 tiles of 16 17.3 / 14.7; top-6, 96 of 8 13.8 / 12.7)
        const bool two = (uint64_t)a.slots * a.up_tiles >= 4ull * device_cus();
        if (packed) return two ? moe_up_launch<T, 2, 1, kMoeOnePacked>(a, a.slots, s) : moe_up_launch<T, 4, 1, kMoeOnePacked>(a, a.slots, s);
        return two ? moe_up_launch<T, 2, 1, kMoeOne>(a, a.slots, s) : moe_up_launch<T, 4, 1, kMoeOne>(a, a.slots, s);
    }
    const dim3 grid(1 + a.x_chunks);
    if (packed) hipLaunchKernelGGL((moe_prepare_kernel<T, true>), grid, dim3(512), 0, s, a);
    else hipLaunchKernelGGL((moe_prepare_kernel<T, false>), grid, dim3(512), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.tokens <= 8) return moe_up_launch<T, 4, 1, kMoePlan>(a, used, s);
    // (us with 2 / 4 waves: 16 tokens, 8 experts of 896 tiles 111 / 114 to 121, 64 of 96, top-6 53.3 / 55.9; 11
    // tokens, 32 of 64 19.4 / 18.5; Q8_0, 16 tokens, 16 of 122 16.2 / 15.7)
    if (a.tokens <= 16)
        return (uint64_t)used * a.up_tiles >= 16ull * device_cus() ? moe_up_launch<T, 2, 2, kMoePlan>(a, used, s)
                                                                   : moe_up_launch<T, 4, 2, kMoePlan>(a, used, s);
    return moe_up_launch<T, 2, 4, kMoePlan>(a, used, s);
}
template <uint32_t T>
static hipError_t moe_down_any(const MoeArgs& a, uint32_t used, hipStream_t s) {
    if (moe_one(a)) return moe_down_launch<T, 16, 1, true>(a, s);
    hipLaunchKernelGGL((moe_h_kernel<T>), dim3(a.h_chunks, used), dim3((a.tokens * 16 + 63) / 64 * 64), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.tokens <= 8) return moe_down_launch<T, 16, 1, false>(a, s);
    if (a.tokens <= 16) return moe_down_launch<T, 12, 2, false>(a, s);
    return moe_down_launch<T, 12, 4, false>(a, s);
}

hipError_t launch_moe_ffn(const MoeCall& c, void* scratch, hipStream_t s) {
    if (c.tokens == 0 || c.slots == 0 || c.experts == 0 || !moe_takes(c)) return hipErrorInvalidValue;
    uint64_t row_bytes = c.cols * 4;  // of x
    if (c.packed) row_bytes = c.up_type == kQ8_0 ? c.cols / 32 * 34 : c.cols / 256 * 292;
    for (uint64_t t0 = 0; t0 < c.tokens; t0 += kMoeTokens) {
        const uint32_t n = c.tokens - t0 < kMoeTokens ? (uint32_t)(c.tokens - t0) : kMoeTokens;
        MoeArgs a{};
        moe_carve(c, n, (uint8_t*)scratch, &a);
        a.tokens = n, a.token0 = (uint32_t)t0, a.slots = (uint32_t)c.slots, a.experts = (uint32_t)c.experts;
        a.cols = (uint32_t)c.cols, a.ffn = (uint32_t)c.ffn, a.out_rows = (uint32_t)c.out_rows;
        a.x = (const uint8_t*)c.x + t0 * row_bytes;
        a.ids = c.ids + t0 * c.slots, a.weights = c.weights + t0 * c.slots;
        a.residual = c.residual ? c.residual + t0 * c.out_rows : nullptr;
        a.y = c.y + t0 * c.out_rows;
        a.gate = c.gate, a.up = c.up, a.down = c.down, a.up_bytes = c.up_bytes, a.down_bytes = c.down_bytes;
        a.up_tiles = (uint32_t)layout_tiles(c.ffn), a.out_tiles = (uint32_t)layout_tiles(c.out_rows);
        a.count = c.count;
        a.x_chunks = (uint32_t)moe_chunks(c.cols), a.h_chunks = (uint32_t)moe_chunks(c.ffn);
        a.x_pairs = (uint32_t)((c.cols / 32 + 1) / 2), a.h_pairs = (uint32_t)((c.ffn / 32 + 1) / 2);
        a.x_row_bytes = layout_chunks_per_tile(c.up_type, c.cols) * layout_chunk_bytes(c.up_type);
        a.h_row_bytes = layout_chunks_per_tile(c.down_type, c.ffn) * layout_chunk_bytes(c.down_type);
        a.err_word = c.err_word;
        const uint64_t pairs = (uint64_t)n * c.slots;
        const uint32_t used = (uint32_t)(pairs < c.experts ? pairs : c.experts);
        hipError_t e = hipErrorInvalidValue;
        switch (c.up_type) {
            case kQ8_0: e = moe_up_any<kQ8_0>(a, c.packed, used, s); break;
            case kQ2_K: e = moe_up_any<kQ2_K>(a, c.packed, used, s); break;
            case kQ3_K: e = moe_up_any<kQ3_K>(a, c.packed, used, s); break;
            case kQ4_K: e = moe_up_any<kQ4_K>(a, c.packed, used, s); break;
            case kQ5_K: e = moe_up_any<kQ5_K>(a, c.packed, used, s); break;
            case kQ6_K: e = moe_up_any<kQ6_K>(a, c.packed, used, s); break;
        }
        if (e != hipSuccess) return e;
        switch (c.down_type) {
            case kQ8_0: e = moe_down_any<kQ8_0>(a, used, s); break;
            case kQ2_K: e = moe_down_any<kQ2_K>(a, used, s); break;
            case kQ3_K: e = moe_down_any<kQ3_K>(a, used, s); break;
            case kQ4_K: e = moe_down_any<kQ4_K>(a, used, s); break;
            case kQ5_K: e = moe_down_any<kQ5_K>(a, used, s); break;
            case kQ6_K: e = moe_down_any<kQ6_K>(a, used, s); break;
            default: e = hipErrorInvalidValue;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace rlq
