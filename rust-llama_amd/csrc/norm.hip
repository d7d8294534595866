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

// Four bytes at any address (a Q8_0 block is 34 bytes long).
struct __attribute__((packed)) Bytes4 {
    uint32_t w;
};

// Four values of a row from element e on; past the end: 0.
template <bool VEC>
__device__ __forceinline__ void norm_load(const float* p, uint32_t e, uint32_t n, float (&v)[4]) {
    if constexpr (VEC) {
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (e < n) f = *(const float4*)(p + e);
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = e + k < n ? p[e + k] : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void norm_store(float* p, uint32_t e, uint32_t n, const float (&v)[4]) {
    if constexpr (VEC) {
        if (e < n) *(float4*)(p + e) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (e + k < n) p[e + k] = v[k];
    }
}

constexpr int kRowShl4 = 0x104;  // lane i <- i + 4 within each 16 lanes

// U Q8_K blocks by a wave, four values of each a lane (the arithmetic of
// rlq_q8k.hpp's q8k_row16; see there for the rounding), of which the first `count`
// exist.  The first value of largest magnitude is that of the first lane that holds
// it, the lanes being in order; the divisions of all blocks run in one go, in a lane
// for each.  The values are finite, or the row is refused anyway.
template <int U>
__device__ __forceinline__ void norm_q8k(const float (&v)[U][4], uint32_t count, NormQ (&o)[U]) {
    const uint32_t lane = threadIdx.x & 63;
    float top = 0.0f;  // lane k: block k's
#pragma unroll
    for (int k = 0; k < U; ++k) {
        float m = v[k][0];
#pragma unroll
        for (int j = 1; j < 4; ++j) m = fabsf(v[k][j]) > fabsf(m) ? v[k][j] : m;
        const uint32_t mag = __float_as_uint(m) & 0x7fffffffu;
        const uint32_t most = wave_max_u32(mag);
        const int first = __builtin_ctzll(__ballot(mag == most));
        const float f = readlane_f(m, first);
        top = lane == (uint32_t)k ? f : top;
    }
    const bool some = top != 0.0f;
    const float inverse = some ? -127.0f / top : 0.0f, d = some ? 1.0f / inverse : 0.0f;
    const unsigned long long bad = __ballot(lane < count && (!finite(inverse) || !finite(d)));
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const float inv = readlane_f(inverse, k);
        uint32_t b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(inv * v[k][j] + 12582912.0f);
        o[k].q = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u) | __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
        o[k].d = readlane_f(d, k);
        int32_t s = dot4(o[k].q, 0x01010101u, 0);
        s += dpp_i<kQuadXor1>(s);
        o[k].bsum = s + dpp_i<kQuadXor2>(s);
        o[k].bad = (bad >> k) & 1;
    }
}

// L lanes per row (four rows share a workgroup of 256 at 64), U times four values per
// lane: lane r holds values 4 (r + k L) .. + 3, so that every load and store of a wave
// is one run of 1 KB.  A row is read once and stays in registers until every check
// of it has passed; then it is written, so a row with a data error keeps its old
// outputs.
//
// The f64 sum runs in a parallel order.  Two orders of the same n nonnegative
// terms differ by at most 2 (n - 1) 2^-53 of their sum, so where both ends of
// that interval give one f32 mean, the reference's mean is that f32 too;
// otherwise (about one row of 4096 values in 65000) the sum is repeated in the
// reference's order.
//
// Bound: memory: 2048 rows of 4096 values into f32 and Q8_K 14.1 us back to back, 5.4 TB/s (20.8
// with sixteen neighbouring values a lane, whose loads and stores touch four times the
// lines); with a residual and its sum 23 us, 6.2 TB/s.  One row: a launch, the loads, two
// barriers and the stores, 4.5 us.
template <int L, int U, bool VEC>
__global__ __launch_bounds__(L < 256 ? 256 : L) void rms_norm_kernel(NormArgs a) {
    constexpr int kWaves = L / 64;  // of a row
    __shared__ double red[kWaves];
    const uint32_t r = threadIdx.x % L, n = a.cols;
    const uint32_t row = blockIdx.x * (L < 256 ? 256 / L : 1) + threadIdx.x / L;
    const bool live = row < a.rows;  // (uniform in a row's lanes)
    const uint64_t at = (uint64_t)(live ? row : 0) * n;
    const float* x = a.x + at;
    const float* res = a.residual ? a.residual + at : nullptr;
    const uint32_t have = live ? n : 0;

    float t[U][4], y[U][4];
#pragma unroll
    for (int k = 0; k < U; ++k) norm_load<VEC>(x, 4 * (r + k * L), have, t[k]);
    if (res) {
#pragma unroll
        for (int k = 0; k < U; ++k) norm_load<VEC>(res, 4 * (r + k * L), have, y[k]);
#pragma unroll
        for (int k = 0; k < U; ++k)
#pragma unroll
            for (int j = 0; j < 4; ++j) t[k][j] = t[k][j] + y[k][j];
    }
#pragma unroll
    for (int k = 0; k < U; ++k) norm_load<VEC>(a.weight, 4 * (r + k * L), n, y[k]);
    double ss = 0.0;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) ss += (double)(t[k][j] * t[k][j]);
    ss = wave_sum_f64(ss);
    if constexpr (L > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) ss += red[w];
    }
    const double dn = (double)n, eps = dn * 2.3e-16 * ss;  // 2^-52 n sum, with a margin
    float mean = (float)(ss / dn);
    if ((float)((ss - eps) / dn) != (float)((ss + eps) / dn)) {  // (uniform in a row's lanes)
        double seq = 0.0;
        if constexpr (L == 64) {
#pragma unroll
            for (int k = 0; k < U; ++k)
                for (uint32_t o = 0; o < 64 && 4 * (o + k * 64) < n; ++o)
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // (past the end: + 0)
                        seq += (double)readlane_f(t[k][j] * t[k][j], (int)o);
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
    bool off = false;  // math.rs:227
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            y[k][j] = t[k][j] * scale * y[k][j];
            off |= !finite(y[k][j]);
        }
    if (live && off) {
        bad = 1;
        report_error(a.err_word, model_key(row, kStFfnNormOut, 0));
    }
    NormQ q[U];
    if (a.q_type) {  // (then n is a multiple of the block, so a block's lanes stay together)
        if (a.q_type == kQ8_K) {
            const uint32_t blocks = have / 256, w = r / 64;  // of the row; the wave's first one
            norm_q8k<U>(y, blocks > w ? (blocks - w + kWaves - 1) / kWaves : 0, q);
        }
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const uint32_t e = 4 * (r + k * L);
            if (e >= have) continue;
            if (a.q_type == kQ8_0) q[k] = norm_q8_0(y[k]);
            if (q[k].bad) {  // (a value that is not finite has been reported above, and sorts first)
                bad = 1;
                report_error(a.err_word, model_key(row, kStGuQuant, e / (a.q_type == kQ8_K ? 256 : 32)));
            }
        }
    }
    if constexpr (L > 64) bad = __syncthreads_or(bad);
    else bad = __ballot(bad) != 0;
    if (bad || !live) return;
    uint8_t* blocks = a.q + ((uint64_t)row * (n / 256) + r / 64) * 292;
#pragma unroll
    for (int k = 0; k < U; ++k) {
        const uint32_t e = 4 * (r + k * L);
        if (e >= n) continue;
        if (a.total) norm_store<VEC>(a.total + at, e, n, t[k]);
        if (a.y) norm_store<VEC>(a.y + at, e, n, y[k]);
        if (a.q_type == kQ8_K) {
            uint8_t* o = blocks + k * (kWaves * 292);
            const uint32_t l = r % 64;
            *(uint32_t*)(o + 4 + 4 * l) = q[k].q;
            // the scale (lane 4) and the sums, two a lane (every eighth)
            const uint32_t next = (uint32_t)dpp_i<kRowShl4>(q[k].bsum);
            const uint32_t pair = ((uint32_t)q[k].bsum & 0xffffu) | next << 16;
            if (l % 8 == 0 || l == 4)
                *(uint32_t*)(o + (l == 4 ? 0 : 260 + l / 2)) = l == 4 ? __float_as_uint(q[k].d) : pair;
        } else if (a.q_type == kQ8_0) {
            uint8_t* o = a.q + (at + e) / 32 * 34;
            const uint32_t l = e / 4 % 8;
            ((Bytes4*)(o + 2 + 4 * l))->w = q[k].q;
            if (l == 0) *(uint16_t*)o = (uint16_t)float_to_half_bits(q[k].d);
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
    const uint32_t fours = (a.cols + 3) / 4;
    if (fours <= 64) return norm_launch<64, 1>(a, vec, s);
    if (fours <= 256) return norm_launch<64, 4>(a, vec, s);
    if (fours <= 512) return norm_launch<256, 2>(a, vec, s);
    if (fours <= 1024) return norm_launch<256, 4>(a, vec, s);
    if (fours <= 2048) return norm_launch<256, 8>(a, vec, s);
    if (fours <= 4096) return norm_launch<1024, 4>(a, vec, s);
    return norm_launch<1024, 8>(a, vec, s);
}

}  // namespace rlq
