// norm.hip - the residual's addition, the RMS norm and its output in 8-bit
// activation blocks on gfx950.
//
// Contract, row by row (crates/model-runtime/src/math.rs:203-228, and the
// quantizers of crates/quant/src/activation.rs:4-51 and encode.rs:79-192):
//   t = x + residual                       (t = x without one)
//   scale = 1 / sqrt(f32(sum t^2 / n) + eps)   squares f32, their sum f64
//   y = t * scale * weight
//   q = the Q8_K or Q8_0 blocks of y
// Every f32 operation rounds as the reference's does, so y and q are the
// reference's bit for bit.
#include "rlq_device.hpp"
#include "rlq_internal.hpp"
#include "rlq_q8k.hpp"

namespace rlq {

// A store of 16 bytes at any address (Q8_0 blocks are 34 bytes long).
struct __attribute__((packed)) Bytes16 {
    uint32_t w[4];
};

// 16 values of a row from element e0 on; past the end: 0.
template <bool VEC>
__device__ __forceinline__ void norm_load(const float* p, uint32_t e0, uint32_t n, float (&v)[16]) {
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (e0 + 4 * k < n) f = *(const float4*)(p + e0 + 4 * k);
            v[4 * k] = f.x, v[4 * k + 1] = f.y, v[4 * k + 2] = f.z, v[4 * k + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = e0 + k < n ? p[e0 + k] : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void norm_store(float* p, uint32_t e0, uint32_t n, const float (&v)[16]) {
    if constexpr (VEC) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e0 + 4 * k < n) *(float4*)(p + e0 + 4 * k) = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    } else {
#pragma unroll
        for (int k = 0; k < 16; ++k)
            if (e0 + k < n) p[e0 + k] = v[k];
    }
}

// L lanes per row (several rows share a workgroup of 256 below 256 lanes), U
// units of 16 values per lane: unit u of the row is lane u % L's number u / L.
// A row is read once and stays in registers until every check of it has passed;
// then it is written, so a row with a data error keeps its old outputs.
//
// The f64 sum runs in a parallel order.  Two orders of the same n nonnegative
// terms differ by at most 2 (n - 1) 2^-53 of their sum, so where both ends of
// that interval give one f32 mean, the reference's mean is that f32 too;
// otherwise (about one row of 4096 values in 65000) the sum is repeated in the
// reference's order.
template <int L, int U, bool VEC>
__global__ __launch_bounds__(L < 256 ? 256 : L) void rms_norm_kernel(NormArgs a) {
    constexpr int kWaves = L / 64;  // of a row, where it has whole waves
    __shared__ double red[L > 64 ? 4 * kWaves : 1];
    const uint32_t r = threadIdx.x % L, n = a.cols, units = (n + 15) / 16;
    const uint32_t row = blockIdx.x * (L < 256 ? 256 / L : 1) + threadIdx.x / L;
    const bool live = row < a.rows;  // (uniform in a row's lanes)
    const uint64_t at = (uint64_t)(live ? row : 0) * n;
    const float* x = a.x + at;
    const float* res = a.residual ? a.residual + at : nullptr;

    float t[U][16], y[U][16];
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const uint32_t e0 = (r + k * L) * 16;
        norm_load<VEC>(x, e0, live ? n : 0, t[k]);
        norm_load<VEC>(a.weight, e0, n, y[k]);
    }
    if (res) {
#pragma unroll
        for (int k = 0; k < U; ++k) {
            float v[16];
            norm_load<VEC>(res, (r + k * L) * 16, live ? n : 0, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) t[k][j] = t[k][j] + v[j];
        }
    }
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int j = 0; j < 16; ++j) ss += (double)(t[k][j] * t[k][j]);
    ss = row16_sum_f64(ss);
    if constexpr (L == 64) ss = rows_sum_f64(ss);
    if constexpr (L > 64) {
        if ((threadIdx.x & 15) == 0) red[threadIdx.x >> 4] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int w = 0; w < 4 * kWaves; ++w) ss += red[w];
    }
    const double dn = (double)n, eps = dn * 2.3e-16 * ss;  // 2^-52 n sum, with a margin
    float mean = (float)(ss / dn);
    if ((float)((ss - eps) / dn) != (float)((ss + eps) / dn)) {  // (uniform in a row's lanes)
        double seq = 0.0;
        if constexpr (L <= 64) {
#pragma unroll
            for (int k = 0; k < U; ++k)
                for (uint32_t o = 0; o < L && o + k * L < units; ++o)
#pragma unroll
                    for (int j = 0; j < 16; ++j) seq += (double)__shfl(t[k][j] * t[k][j], (int)o, L);
        } else {
            __syncthreads();  // every thread has read red[]
            if (threadIdx.x < 64) {
                for (uint32_t i = 0; i < n; i += 64) {
                    const uint32_t e = i + threadIdx.x;
                    float v = 0.0f;
                    if (e < n) v = res ? x[e] + res[e] : x[e];
                    v = v * v;
                    const uint32_t m = n - i < 64 ? n - i : 64;
                    for (uint32_t l = 0; l < m; ++l) seq += (double)readlane_f(v, (int)l);
                }
                if (threadIdx.x == 0) red[0] = seq;
            }
            __syncthreads();
            seq = red[0];
        }
        mean = (float)(seq / dn);
    }
    const float scale = 1.0f / sqrtf(mean + a.eps);
    int bad = 0;
    if (live && (!(scale <= 3.402823466e38f) || !(scale > 0.0f))) {  // math.rs:218-220
        bad = 1;
        if (r == 0) report_error(a.err_word, model_key(row, kStFfnNormScale, 0));
    }
    uint32_t q[U][4];
    float d[U];
    int32_t bsum[U];
    bool off = false;  // math.rs:227
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            y[k][j] = t[k][j] * scale * y[k][j];
            off |= !finite(y[k][j]);
        }
    if (live && off) {
        bad = 1;
        report_error(a.err_word, model_key(row, kStFfnNormOut, 0));
    }
    if (a.q_type) {  // (then n is a multiple of the block, so a block's lanes stay together)
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint32_t u = r + k * L;
            if (!live || u >= units) continue;
            int kind;
            if (a.q_type == kQ8_K) {
                const Q8KRow o = q8k_row16(y[k], u & 15);
#pragma unroll
                for (int w = 0; w < 4; ++w) q[k][w] = o.q[w];
                d[k] = o.d, bsum[k] = o.bsum, kind = o.kind;
            } else {
                uint32_t index;
                kind = q8_0_pair16(y[k], u & 1, q[k], d[k], index);
            }
            if (kind >= 0) {  // a non-finite value has been reported above, and sorts first
                bad = 1;
                if (kind == kKindScale)
                    report_error(a.err_word, model_key(row, kStGuQuant, u / (a.q_type == kQ8_K ? 16 : 2)));
            }
        }
    }
    if constexpr (L > 64) {
        bad = __syncthreads_or(bad);
    } else {
        const unsigned long long m = __ballot(bad);
        bad = L == 64 ? m != 0 : ((m >> (threadIdx.x & 48)) & 0xffffull) != 0;
    }
    if (bad || !live) return;
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const uint32_t u = r + k * L, e0 = u * 16;
        if (u >= units) continue;
        if (a.total) norm_store<VEC>(a.total + at, e0, n, t[k]);
        if (a.y) norm_store<VEC>(a.y + at, e0, n, y[k]);
        if (a.q_type == kQ8_K) {
            uint8_t* o = a.q + ((uint64_t)row * (n / 256) + u / 16) * 292;
            if ((u & 15) == 0) *(float*)o = d[k];
            *(Bytes16*)(o + 4 + 16 * (u & 15)) = Bytes16{{q[k][0], q[k][1], q[k][2], q[k][3]}};
            *(int16_t*)(o + 260 + 2 * (u & 15)) = (int16_t)bsum[k];
        } else if (a.q_type == kQ8_0) {
            uint8_t* o = a.q + ((uint64_t)row * (n / 32) + u / 2) * 34;
            // d is the f32 of a half: converting it back is exact
            if ((u & 1) == 0) *(uint16_t*)o = (uint16_t)float_to_half_bits(d[k]);
            *(Bytes16*)(o + 2 + 16 * (u & 1)) = Bytes16{{q[k][0], q[k][1], q[k][2], q[k][3]}};
        }
    }
}

template <int L, int U>
static hipError_t norm_launch(const NormArgs& a, bool vec, hipStream_t s) {
    constexpr uint32_t per = L < 256 ? 256 / L : 1;
    const dim3 grid((a.rows + per - 1) / per), block(L < 256 ? 256 : L);
    if (vec) hipLaunchKernelGGL((rms_norm_kernel<L, U, true>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((rms_norm_kernel<L, U, false>), grid, block, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_rms_norm(const NormArgs& a, hipStream_t s) {
    if (a.rows == 0 || a.cols == 0 || a.cols > kNormMaxCols) return hipErrorInvalidValue;
    uintptr_t low = (uintptr_t)a.x | (uintptr_t)a.residual | (uintptr_t)a.weight | (uintptr_t)a.total | (uintptr_t)a.y;
    const bool vec = (low & 15) == 0 && a.cols % 4 == 0;
    const uint32_t units = (a.cols + 15) / 16;
    if (units <= 16) return norm_launch<16, 1>(a, vec, s);
    if (units <= 64) return norm_launch<64, 1>(a, vec, s);
    if (units <= 256) return norm_launch<256, 1>(a, vec, s);
    if (units <= 512) return norm_launch<256, 2>(a, vec, s);
    if (units <= 1024) return norm_launch<1024, 1>(a, vec, s);
    return norm_launch<1024, 2>(a, vec, s);
}

}  // namespace rlq
