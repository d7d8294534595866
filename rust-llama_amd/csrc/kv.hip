// kv.hip - a paged KV cache on gfx950: pages off a free list, the store of rotated
// keys and of values, attention of new tokens over the pages, and the beams' tables.
//
// A cache's layer holds, for each page and KV head, a plane of `page` tokens:
// token after token their `dim` values (f32, f16, bf16), or (Q8_0) their levels and
// after those, token after token, the f16 scales of their blocks of 32.
#include "rlq_device.hpp"
#include "rlq_internal.hpp"
#include "rlq_q8k.hpp"

namespace rlq {

// ---------------------------------------------------------------------------
// Pages of the requests
// ---------------------------------------------------------------------------

// Why a request gets no pages (rlq.h, RLQ_INVALID_STATE of rlq_kv_pages).
enum PagesRefusal : uint32_t { kBadCount = 0, kNoPage = 1, kNoColumn = 2, kNoRow = 3, kBadLength = 4 };

// Three sums over the threads before this one, and over all.
template <uint32_t N>
__device__ __forceinline__ void plan_scan(uint64_t (&v)[3], uint64_t (&total)[3], uint64_t (*part)[3]) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t sum[3] = {v[0], v[1], v[2]};
    for (int m = 1; m < 64; m <<= 1) {
        uint64_t o[3];
#pragma unroll
        for (int k = 0; k < 3; ++k) o[k] = __shfl_up(sum[k], m, 64);
#pragma unroll
        for (int k = 0; k < 3; ++k) sum[k] += (int)lane >= m ? o[k] : 0;
    }
    if (lane == 63)
        for (int k = 0; k < 3; ++k) part[wave][k] = sum[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        uint64_t before = 0;
        total[k] = 0;
        for (uint32_t w = 0; w < N / 64; ++w) {
            const uint64_t p = part[w][k];
            before += w < wave ? p : 0;
            total[k] += p;
        }
        v[k] = before + sum[k] - v[k];
    }
}

// The last of the n + 1 ascending numbers that is not above v (at[0] = 0 <= v < at[n]).
template <class P>
__device__ __forceinline__ uint32_t segment_of(const P* at, uint32_t n, uint32_t v) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if ((uint32_t)at[mid] <= v) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Row t of the batch: its request, position and slot; -1 behind the last.  after: the
// requests' lengths with their new tokens.
template <class P>
__device__ __forceinline__ void pages_row(const PagesArgs& a, const P* starts, uint32_t total, uint32_t t, const int32_t* after) {
    int32_t request = -1, position = -1;
    int64_t slot = -1;
    if (t < total) {
        const uint32_t r = segment_of(starts, a.requests, t);
        const uint32_t ahead = (uint32_t)starts[r + 1] - t;  // rows of the request from this one on
        request = (int32_t)r;
        position = after[r] - (int32_t)ahead;
        const int32_t page = a.tables[(uint64_t)r * a.width + ((uint32_t)position >> a.log_page)];
        // (no page: no slot that a store would take or leave alone)
        slot = page < 0 ? -2 : ((int64_t)page << a.log_page) + (position & ((1 << a.log_page) - 1));
    }
    a.out_requests[t] = request;
    a.positions[t] = position;
    a.slots[t] = slot;
}

// One workgroup: sums over the requests, the ended requests' pages onto the free
// list, pages off its top (request after request, the t-th from the top is the t-th
// page taken), and, where `rows`, the batch's rows.  Everything is checked before
// anything is written.
//
// N threads, PER requests each.
//
// Bound: latencies one after another (the lengths, the ended requests' entries, the list, the tables) and the
// barriers between: 32 requests of up to 8192 tokens, one new token each, a tenth of them ended, 6.2 us (11.6 with
// the entries loaded 64 at a time); 256 requests that take 2000 pages 9.8, and their 65536 rows 3.8 in a launch of
// their own.
template <uint32_t N, uint32_t PER>
__global__ __launch_bounds__(N) void pages_plan_kernel(PagesArgs a, uint32_t rows) {
    constexpr uint32_t kMost = N * PER, kWaves = N / 64;
    __shared__ uint64_t part[kWaves][3];
    __shared__ uint32_t need[kMost + 1], start[kMost + 1], gone[kMost];
    __shared__ int32_t later[kMost];
    __shared__ uint16_t ended[kMost];
    __shared__ uint32_t n_ended, first_bad;
    __shared__ unsigned long long bad_page;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.requests;
    const int64_t free0 = *a.count;
    if (tid == 0) n_ended = 0, first_bad = 0xffffffffu, bad_page = ~0ull;
    // a request's columns of the table in use, the pages and the rows it gets
    int32_t before[PER], more[PER];
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t r = tid * PER + i;
        before[i] = r < n ? a.before[r] : 0;
        more[i] = r < n ? a.more[r] : 0;
    }
    __syncthreads();

    uint32_t refused = 0xffffffffu;  // request * 8 + the reason
    auto refuse = [&](uint32_t r, uint32_t why) { refused = r * 8 + why < refused ? r * 8 + why : refused; };
    auto held = [&](int64_t len) { return (uint64_t)(len + (1 << a.log_page) - 1) >> a.log_page; };
    uint64_t sums[3] = {}, totals[3];  // pages, rows, pages that come back
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t r = tid * PER + i;
        const int64_t after = (int64_t)before[i] + (more[i] > 0 ? more[i] : 0);
        if (before[i] < 0 || after > 0x7fffffff || held(after) > a.width) {
            refuse(r, before[i] < 0 || after > 0x7fffffff ? kBadLength : kNoColumn);
            before[i] = more[i] = 0;
        }
        if (r < n) {
            gone[r] = 0;
            if (more[i] < 0 && before[i]) ended[atomicAdd(&n_ended, 1u)] = (uint16_t)r;
        }
        if (more[i] > 0) sums[0] += held(after) - held(before[i]), sums[1] += (uint32_t)more[i];
    }
    __syncthreads();
    // a wave per ended request, 512 of its entries at a time
    auto entries = [&](uint32_t r, auto&& take) {
        const uint64_t row = (uint64_t)r * a.width;
        const uint32_t cols = (uint32_t)held(a.before[r]);
        for (uint32_t c = lane; c < cols + lane; c += 512) {
            int32_t p[8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) p[k] = c + 64 * k < cols ? a.owned[row + c + 64 * k] : -1;
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) take(row + c + 64 * k, p[k]);
        }
    };
    for (uint32_t i = wave; i < n_ended; i += kWaves) {
        uint32_t some = 0;
        entries(ended[i], [&](uint64_t at, int32_t p) {
            if (p >= 0 && (uint32_t)p >= a.pages) atomicMin(&bad_page, (unsigned long long)at);
            some += (uint32_t)__builtin_popcountll(__ballot(p >= 0));
        });
        if (lane == 0) gone[ended[i]] = some;
    }
    if (n_ended) __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i)
        if (tid * PER + i < n) sums[2] += gone[tid * PER + i];
    plan_scan<N>(sums, totals, part);
    const bool sound = free0 >= 0 && free0 <= (int64_t)a.pages && (uint64_t)free0 + totals[2] <= a.pages;
    const uint64_t top = (sound ? (uint64_t)free0 : 0) + totals[2];
    if (!sound) refuse(0, kBadCount);
    auto cut = [](uint64_t v) { return (uint32_t)(v < 0xffffffffull ? v : 0xffffffffull); };
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t r = tid * PER + i;
        if (r >= n) break;
        const int64_t after = (int64_t)before[i] + (more[i] > 0 ? more[i] : 0);
        need[r] = cut(sums[0]);
        start[r] = cut(sums[1]);
        later[r] = more[i] < 0 ? 0 : (int32_t)after;
        const uint32_t g = gone[r];
        gone[r] = cut(sums[2]);
        sums[2] += g;
        if (more[i] > 0) sums[0] += held(after) - held(before[i]), sums[1] += (uint32_t)more[i];
        if (sums[0] > top) refuse(r, kNoPage);
        if (sums[1] > a.tokens) refuse(r, kNoRow);
    }
    if (refused != 0xffffffffu) atomicMin(&first_bad, refused);
    const uint32_t total_need = (uint32_t)totals[0], total_rows = (uint32_t)totals[1];  // (within 32 bits, or refused)
    if (tid == 0) need[n] = total_need, start[n] = total_rows;
    __syncthreads();
    const bool bad = first_bad != 0xffffffffu || bad_page != ~0ull;
    if (tid == 0) {
        *a.refused = bad;
        if (bad_page != ~0ull) report_error(a.err_word, bounds_key(bad_page));
        else if (bad) report_error(a.err_word, model_key(first_bad / 8, kStPages, first_bad % 8));
    }
    if (bad) return;

    for (uint32_t i = wave; i < n_ended; i += kWaves) {
        uint64_t to = (uint64_t)free0 + gone[ended[i]];
        entries(ended[i], [&](uint64_t at, int32_t p) {
            const unsigned long long m = __ballot(p >= 0);
            if (p >= 0) {
                a.free[to + __builtin_popcountll(m & ((1ull << lane) - 1))] = p;
                a.owned[at] = -1;
            }
            to += __builtin_popcountll(m);
        });
    }
    if (n_ended) __syncthreads();
    for (uint32_t t = tid; t < total_need; t += N) {
        const uint32_t r = segment_of(need, n, t);
        // (a request's last new page is that of its last token)
        const uint64_t at = (uint64_t)r * a.width + held(later[r]) - (need[r + 1] - t);
        const int32_t p = a.free[top - 1 - t];
        a.tables[at] = p;
        if (a.owned != a.tables) a.owned[at] = p;
    }
    if (n_ended || rows) __syncthreads();  // (the lengths may take the place of `before`; the rows read the tables)
#pragma unroll
    for (uint32_t i = 0; i < PER; ++i) {
        const uint32_t r = tid * PER + i;
        if (r >= n) break;
        a.after[r] = later[r];
        a.starts[r] = (int32_t)start[r];
    }
    if (tid == 0) a.starts[n] = (int32_t)total_rows, *a.count_after = (int32_t)(top - total_need);
    if (!rows) return;
    for (uint32_t t = tid; t < a.tokens; t += N) pages_row(a, start, total_rows, t, later);
}

__global__ __launch_bounds__(256) void pages_rows_kernel(PagesArgs a) {
    __shared__ int32_t starts[kKvMaxRequests + 1];
    for (uint32_t r = threadIdx.x; r <= a.requests; r += 256) starts[r] = a.starts[r];
    const uint32_t refused = *a.refused;
    __syncthreads();
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;
    if (t < a.tokens && !refused) pages_row(a, starts, (uint32_t)starts[a.requests], t, a.after);
}

hipError_t launch_kv_pages(const PagesArgs& a, hipStream_t s) {
    if (a.requests == 0 || a.requests > kKvMaxRequests || a.tokens > 0x7fffffffu) return hipErrorInvalidValue;
    // one workgroup writes 4096 rows in the time of another launch (four rounds of 1024 threads); few requests and
    // rows: a small workgroup, whose barriers and sums are cheaper (32 requests 6.2 us, 7.0 with 1024 threads)
    const bool one = a.tokens <= 4096;
    if (a.requests <= 256 && a.tokens <= 1024)
        hipLaunchKernelGGL((pages_plan_kernel<256, 1>), dim3(1), dim3(256), 0, s, a, 1u);
    else if (a.requests <= 1024)
        hipLaunchKernelGGL((pages_plan_kernel<1024, 1>), dim3(1), dim3(1024), 0, s, a, one ? 1u : 0u);
    else
        hipLaunchKernelGGL((pages_plan_kernel<1024, kKvMaxRequests / 1024>), dim3(1), dim3(1024), 0, s, a, one ? 1u : 0u);
    if (!one) hipLaunchKernelGGL(pages_rows_kernel, dim3((a.tokens + 255) / 256), dim3(256), 0, s, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Store
// ---------------------------------------------------------------------------

template <uint32_t T>
__device__ __forceinline__ uint64_t kv_row(uint32_t dim) {  // bytes of a token's values (Q8_0: levels) in a plane
    return T == kQ8_0 ? dim : T == kF32 ? 4 * dim : 2 * dim;
}
template <uint32_t T>
__device__ __forceinline__ uint64_t kv_plane(uint32_t dim, uint32_t log_page) {
    return (T == kQ8_0 ? dim + dim / 16 : kv_row<T>(dim)) << log_page;
}

__device__ __forceinline__ uint32_t bf16_bits(float v) {  // ties to even; v is finite
    const uint32_t b = __float_as_uint(v);
    return (b + 0x7fffu + ((b >> 16) & 1)) >> 16;
}

// N words at an address that is a multiple of A bytes.
template <class W, int N, int A>
struct __attribute__((packed, aligned(A))) Words {
    W w[N];
};
template <class W, int N, int A>
__device__ __forceinline__ void words(const void* p, W (&out)[N]) {
    const Words<W, N, A> t = *(const Words<W, N, A>*)p;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = t.w[i];
}
// sine and cosine of a by quarter turns: a - n pi/2 with pi/2 in two f64 (n below 2^38, so that what is
// left out, n 2^-108, is far below a last bit), then the Taylor polynomials, whose
// first terms left out are below 2^-63 (sine) and 2^-58 (cosine) for |r| <= pi/4.
__device__ __forceinline__ double2 sine_cosine(double a) {
    if (!(fabs(a) < 2.7e11)) {
        double s, c;
        sincos(a, &s, &c);
        return make_double2(s, c);
    }
    const double n = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.5707963267948965580, a);
    r = __builtin_fma(-n, 6.1232339957367660359e-17, r);
    const double z = r * r;
    double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;  // 1 / 17!, 1 / 16!
    s = __builtin_fma(s, z, -1.0 / 1307674368000.0);
    c = __builtin_fma(c, z, -1.0 / 87178291200.0);
    s = __builtin_fma(s, z, 1.0 / 6227020800.0);
    c = __builtin_fma(c, z, 1.0 / 479001600.0);
    s = __builtin_fma(s, z, -1.0 / 39916800.0);
    c = __builtin_fma(c, z, -1.0 / 3628800.0);
    s = __builtin_fma(s, z, 1.0 / 362880.0);
    c = __builtin_fma(c, z, 1.0 / 40320.0);
    s = __builtin_fma(s, z, -1.0 / 5040.0);
    c = __builtin_fma(c, z, -1.0 / 720.0);
    s = __builtin_fma(s, z, 1.0 / 120.0);
    c = __builtin_fma(c, z, 1.0 / 24.0);
    s = __builtin_fma(s, z, -1.0 / 6.0);
    c = __builtin_fma(c, z, -0.5);
    s = __builtin_fma(s * z, r, r);
    c = __builtin_fma(c, z, 1.0);
    const int64_t q = (int64_t)n;
    const double u = q & 1 ? c : s, v = q & 1 ? s : c;
    return make_double2(q & 2 ? -u : u, (q + 1) & 2 ? -v : v);
}

// Whether a stored value would be no finite number of the cache's type.
template <uint32_t T>
__device__ __forceinline__ bool store_off(float y) {
    if constexpr (T == kF16) return !finite((float)(_Float16)y);
    if constexpr (T == kBF16) return !finite(y) || !finite(__uint_as_float(bf16_bits(y) << 16));
    return !finite(y);
}
// The first such of four values, of which one is; q: of a query's, which are not stored.
template <uint32_t T>
__device__ __forceinline__ uint32_t first_off(const float (&y)[4], bool q) {
    uint32_t first = 3;
#pragma unroll
    for (int j = 2; j >= 0; --j)
        if (q ? !finite(y[j]) : store_off<T>(y[j])) first = (uint32_t)j;
    return first;
}
// Four values from element e on of a token's place in a plane; Q8_0: by eight lanes, a block.
template <uint32_t T>
__device__ __forceinline__ void store_put(uint8_t* plane, uint64_t row, uint32_t e, uint32_t dim, uint32_t log_page,
                                          const float (&y)[4]) {
    uint8_t* to = plane + row * kv_row<T>(dim);
    if constexpr (T == kF32) {
        *(float4*)(to + 4 * e) = make_float4(y[0], y[1], y[2], y[3]);
    } else if constexpr (T == kQ8_0) {
        const NormQ q = norm_q8_0(y);
        *(uint32_t*)(to + e) = q.q;
        if (e % 32 == 0)
            *(uint16_t*)(plane + ((uint64_t)dim << log_page) + 2 * (row * (dim / 32) + e / 32)) = (uint16_t)float_to_half_bits(q.d);
    } else {
        uint32_t b[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
            b[j] = T == kF16 ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)y[j]) : bf16_bits(y[j]);
        *(uint2*)(to + 2 * e) = make_uint2(b[0] | b[1] << 16, b[2] | b[3] << 16);
    }
}

// A token's query, key and value heads.  The first 2 * half values of a query or key head are
// rotated:
//   (x, y) -> (x cos a - y sin a, x sin a + y cos a),  a = position * freq[i]
// of neighbours (pairs) or of values half apart; angle, sine, cosine, products and sum in
// f64, rounded once to f32, so that the stored 16 bits and levels are defined to the last
// one.
//
// A workgroup of N threads per token, a thread U times four values.  All are loaded, with their partners,
// before the angles are made and stored after every one has been checked: a token with an
// error keeps its place, and q_out may be q.  Needs whole fours of rotated values (half a
// multiple of 4, of pairs 2).
//
// Bound: one token: a launch, one round of loads, two barriers, 4.7 us (10.6 with loads for the check and again
// for the store, angles before them and a library's sine); 1777 tokens of 14 query and 2 KV heads of 64 into Q8_0
// 9.0 us for 15 MB: f64 rotation and the quantizer beside one round of latencies.
template <uint32_t T, int N, int U>
__global__ __launch_bounds__(N) void kv_store_kernel(StoreArgs a) {
    __shared__ double2 turn[128];  // cosine, sine
    const uint32_t tid = threadIdx.x, dim = a.c.dim, L = dim / 4, kv = a.c.kv_heads, units = (a.heads + 2 * kv) * L;
    const uint64_t t = blockIdx.x;
    const int64_t slot = a.slots[t];
    const uint32_t magic = 0xffffffffu / L + 1;  // x / L = x magic >> 32 for x below 2^26
    float x[U][4], o[U][4];
    uint32_t head[U], e[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t i = tid + N * u < units ? tid + N * u : units - 1;
        head[u] = __umulhi(i, magic);
        e[u] = 4 * (i - head[u] * L);
        const bool q = head[u] < a.heads, k = head[u] < a.heads + kv;
        const float* p = q ? a.q + t * a.q_stride + (uint64_t)head[u] * dim
                           : k ? a.k + t * a.k_stride + (uint64_t)(head[u] - a.heads) * dim
                               : a.v + t * a.v_stride + (uint64_t)(head[u] - a.heads - kv) * dim;
        words<float, 4, 4>(p + e[u], x[u]);
        const bool turns = k && e[u] < 2 * a.half;
        if (!a.pairs && turns) words<float, 4, 4>(p + (e[u] < a.half ? e[u] + a.half : e[u] - a.half), o[u]);
        else o[u][0] = x[u][1], o[u][1] = x[u][0], o[u][2] = x[u][3], o[u][3] = x[u][2];
    }
    if (slot == -1) return;  // a row behind the batch's last
    if (slot < 0 || (uint64_t)slot >= a.c.pages << a.c.log_page) {
        if (tid == 0) report_error(a.err_word, bounds_key(t));
        return;
    }
    if (tid < a.half) {
        const double2 sc = sine_cosine((double)a.positions[t] * (double)a.freqs[tid]);
        turn[tid] = make_double2(sc.y, sc.x);
    }
    __syncthreads();
    int bad = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool q = head[u] < a.heads, k = head[u] < a.heads + kv, have = tid + N * u < units;
        if (k && e[u] < 2 * a.half) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) {
                const uint32_t i = e[u] + j;
                const bool second = a.pairs ? j & 1 : i >= a.half;
                const double2 cs = turn[a.pairs ? i / 2 : second ? i - a.half : i];
                const double m = (double)x[u][j] * cs.x, r = (double)o[u][j] * cs.y;
                x[u][j] = (float)(second ? r + m : m - r);
            }
        }
        bool off = false;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) off |= q ? !finite(x[u][j]) : store_off<T>(x[u][j]);
        bool scale = false;
        if constexpr (T == kQ8_0) scale = !q && norm_q8_0(x[u]).bad;
        if (have && (off || scale)) {
            bad = 1;
            const uint64_t at = (uint64_t)head[u] * dim + e[u];
            report_error(a.err_word, off ? error_key(t, kKindNonFinite, at + first_off<T>(x[u], q))
                                         : error_key(t, kKindScale, (at - (uint64_t)a.heads * dim) / 32));
        }
    }
    if (__syncthreads_or(bad)) return;
    const uint64_t page = (uint64_t)slot >> a.c.log_page, row = (uint64_t)slot & ((1u << a.c.log_page) - 1);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (tid + N * u >= units) continue;
        if (head[u] < a.heads) {
            Words<float, 4, 4> y{{x[u][0], x[u][1], x[u][2], x[u][3]}};
            *(Words<float, 4, 4>*)(a.q_out + t * a.out_stride + (uint64_t)head[u] * dim + e[u]) = y;
        } else {
            const uint32_t g = head[u] - a.heads;
            uint8_t* base = g < kv ? a.c.k + page * a.c.k_stride : a.c.v + page * a.c.v_stride;
            store_put<T>(base + (g < kv ? g : g - kv) * kv_plane<T>(dim, a.c.log_page), row, e[u], dim, a.c.log_page, x[u]);
        }
    }
}

// The same for any half and number of heads: dim / 4 lanes a head, a wave whole heads at a time, which it loads
// before it stores them; the values are made twice, to be checked and to be stored.
template <uint32_t T>
__global__ __launch_bounds__(256) void kv_store_any_kernel(StoreArgs a) {
    __shared__ double2 turn[128];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, dim = a.c.dim;
    const uint64_t t = blockIdx.x;
    const int64_t slot = a.slots[t];
    if (slot == -1) return;  // a row behind the batch's last
    if (slot < 0 || (uint64_t)slot >= a.c.pages << a.c.log_page) {
        if (threadIdx.x == 0) report_error(a.err_word, bounds_key(t));
        return;
    }
    if (threadIdx.x < a.half) {
        const double2 sc = sine_cosine((double)a.positions[t] * (double)a.freqs[threadIdx.x]);
        turn[threadIdx.x] = make_double2(sc.y, sc.x);
    }
    __syncthreads();
    const uint32_t L = dim / 4, per = 64 / L, group = lane / L, e = 4 * (lane % L);
    const uint32_t kv = a.c.kv_heads, heads = a.heads + 2 * kv;
    const uint64_t page = (uint64_t)slot >> a.c.log_page, row = (uint64_t)slot & ((1u << a.c.log_page) - 1);

    // four values of head h, and whether one is not finite
    auto values = [&](uint32_t h, float (&y)[4]) {
        const bool q = h < a.heads, k = !q && h < a.heads + kv;
        const float* x = q ? a.q + t * a.q_stride + (uint64_t)h * dim
                           : k ? a.k + t * a.k_stride + (uint64_t)(h - a.heads) * dim
                               : a.v + t * a.v_stride + (uint64_t)(h - a.heads - kv) * dim;
        bool off = false;
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            const uint32_t i = e + j;
            y[j] = x[i];
            if ((q || k) && i < 2 * a.half) {
                const bool second = a.pairs ? i & 1 : i >= a.half;
                const uint32_t other = a.pairs ? i ^ 1 : second ? i - a.half : i + a.half;
                const double2 cs = turn[a.pairs ? i / 2 : second ? i - a.half : i];
                const double m = (double)y[j] * cs.x, o = (double)x[other] * cs.y;
                y[j] = (float)(second ? o + m : m - o);
            }
            off |= q ? !finite(y[j]) : store_off<T>(y[j]);
        }
        return off;
    };

    int bad = 0;
    for (uint32_t h = wave * per + group; h < heads && group < per; h += 4 * per) {
        float y[4];
        if (values(h, y)) {
            bad = 1;
            report_error(a.err_word, error_key(t, kKindNonFinite, (uint64_t)h * dim + e + first_off<T>(y, h < a.heads)));
        } else if (T == kQ8_0 && h >= a.heads && norm_q8_0(y).bad) {
            bad = 1;
            report_error(a.err_word, error_key(t, kKindScale, ((uint64_t)(h - a.heads) * dim + e) / 32));
        }
    }
    if (__syncthreads_or(bad)) return;
    for (uint32_t h = wave * per + group; h < heads && group < per; h += 4 * per) {
        float y[4];
        values(h, y);
        if (h < a.heads) {
            float* out = a.q_out + t * a.out_stride + (uint64_t)h * dim + e;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) out[j] = y[j];
            continue;
        }
        const uint32_t g = h - a.heads < kv ? h - a.heads : h - a.heads - kv;
        uint8_t* plane = (h - a.heads < kv ? a.c.k + page * a.c.k_stride : a.c.v + page * a.c.v_stride) +
                         g * kv_plane<T>(dim, a.c.log_page);
        store_put<T>(plane, row, e, dim, a.c.log_page, y);
    }
}

template <uint32_t T>
static hipError_t store_launch(const StoreArgs& a, hipStream_t s) {
    const uint64_t units = (uint64_t)(a.heads + 2 * a.c.kv_heads) * (a.c.dim / 4);
    const dim3 grid((uint32_t)a.tokens);
    // few tokens: large workgroups, one or two fours a thread
    const bool few = a.tokens <= (uint64_t)device_cus(), whole = a.half % (a.pairs ? 2 : 4) == 0;
    if (!whole || units > (few ? 4096 : 2048)) hipLaunchKernelGGL(kv_store_any_kernel<T>, grid, dim3(256), 0, s, a);
    else if (few && units <= 1024) hipLaunchKernelGGL((kv_store_kernel<T, 1024, 1>), grid, dim3(1024), 0, s, a);
    else if (few && units <= 2048) hipLaunchKernelGGL((kv_store_kernel<T, 1024, 2>), grid, dim3(1024), 0, s, a);
    else if (few) hipLaunchKernelGGL((kv_store_kernel<T, 1024, 4>), grid, dim3(1024), 0, s, a);
    else if (units <= 512) hipLaunchKernelGGL((kv_store_kernel<T, 256, 2>), grid, dim3(256), 0, s, a);
    else if (units <= 1024) hipLaunchKernelGGL((kv_store_kernel<T, 256, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_store_kernel<T, 256, 8>), grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_kv_store(const StoreArgs& a, hipStream_t s) {
    if (a.tokens == 0 || a.tokens > 0x7fffffffu || a.c.dim % 32 || a.c.dim > 256 || 2 * a.half > a.c.dim)
        return hipErrorInvalidValue;
    switch (a.c.type) {
        case kF32: return store_launch<kF32>(a, s);
        case kF16: return store_launch<kF16>(a, s);
        case kBF16: return store_launch<kBF16>(a, s);
        case kQ8_0: return store_launch<kQ8_0>(a, s);
        default: return hipErrorInvalidValue;
    }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int pow2_of(int n) { return n & -n; }

__device__ __forceinline__ f32x4 mma_f16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma_bf16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// An f32 number as 16-bit terms: two f16, each to nearest, whose sum it is to 23 bits (queries and weights begin near f16's
// upper end; below 2^-16 of the largest the lower term's least step, 2^-24, ends the number earlier, which is then off by
// 2^-38 of the largest at most), or three bf16, whose sum it is to its last bit.  To nearest, because what is cut off towards
// zero adds up: 20000 small weights were 1.4e-3 of their sum low.
// The terms of eight numbers, as operands.
__device__ __forceinline__ void split_f16(const float (&x)[8], uint32_t (&hi)[4], uint32_t (&lo)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 h = __builtin_convertvector((f32x2{x[2 * i], x[2 * i + 1]}), f16x2);
        hi[i] = __builtin_bit_cast(uint32_t, h);
        const f32x2 r = {x[2 * i] - (float)h[0], x[2 * i + 1] - (float)h[1]};
        lo[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, f16x2));
    }
}
__device__ __forceinline__ void split_bf16(const float (&x)[8], uint32_t (&hi)[4], uint32_t (&mid)[4], uint32_t (&lo)[4]) {
    uint32_t t[3][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t[0][i] = __float_as_uint(x[i]);
        const float r = x[i] - __uint_as_float(t[0][i] & 0xffff0000u);
        t[1][i] = __float_as_uint(r);
        t[2][i] = __float_as_uint(r - __uint_as_float(t[1][i] & 0xffff0000u));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // the upper halves of two
        hi[i] = __builtin_amdgcn_perm(t[0][2 * i + 1], t[0][2 * i], 0x07060302u);
        mid[i] = __builtin_amdgcn_perm(t[1][2 * i + 1], t[1][2 * i], 0x07060302u);
        lo[i] = __builtin_amdgcn_perm(t[2][2 * i + 1], t[2][2 * i], 0x07060302u);
    }
}

// The maximum and the sum over the lanes 16 apart; every lane gets it.
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// A wave's part of the attention of up to 16 query heads (columns) over the tokens of one
// KV head, 32 tokens at a time (two halves of 16).
//
//   S = K Q    v_mfma_f32_16x16x32 (f32: 16x16x4): rows are tokens, columns query heads.
//              Lane (i, g) = (lane % 16, lane / 16) loads 16 bytes of token i.
//   O = V^T P  rows are values, columns query heads.  Lane (i, g) gets from S the scores of
//              tokens 4g .. 4g + 3 of each half for head i, which are its operand of P as they are;
//              it loads dim / 16 values of these eight tokens, values i * dim / 16 and on, and pairs
//              of tokens are put together in registers (one v_perm a pair).
//
// Neither goes through LDS.  The scores' operands and P are f32 numbers in 16-bit terms (split_*),
// so the products are those of f32 (with f16 terms of 23 bits) with the stored values; the matrix cores have room for that:
// 16-bit keys and values need 2 (f16) or 3 (bf16) times 256 cycles per 32 tokens of 128 values, of
// about 1900 that HBM takes for them (one SIMD's share).  Q8_0: scores with f16 levels, block by block, times
// the block's scale; a value, level times scale, as the sum of two f16, which holds it exactly: a product of 18
// bits that is a multiple of 2^-24, -128 times a scale of 511.75 at most, which is f16's largest (with a larger scale
// among them the 32 tokens take f32 values on 16x16x4, 2048 cycles of the matrix cores instead of 384).  Of the four
// products of a weight's and a value's terms the lower two's is left out: 2^-22 of the whole at most, of either sign, about one
// rounding of f32 in the mean square (with it 32 rows of 4096 tokens take 59.6 us instead of 59.0, five drafted rows each 108
// instead of 106).
// Blocks of 32 values to which two workgroups' registers fit a CU (a wave's tile, queries and
// accumulators, 256 of them).
constexpr uint32_t attn_wide(uint32_t type) { return type == kF32 ? 3 : 4; }

template <uint32_t T, int NB>  // NB: blocks of 32 values
struct AttnWave {
    static constexpr int kDim = 32 * NB, kOwn = 2 * NB;  // values of a token that a lane holds for O
    static constexpr bool k16 = T == kF16 || T == kBF16;
    // Weights are exp(s - max) times kTop.  (In the exponent it would be rounded with the maximum: weights of scores up to 16 off
    // by 3e-7 among the waves, rows of four tokens by 1.6e-7 instead of 1.0e-7, and one token's weight not 1.)
    static constexpr float kTop = T == kF16 || T == kQ8_0 ? 16384.0f : 1.0f;

    // q (columns past the last head 0): f32, or in terms
    uint32_t q0[T == kF32 ? 1 : NB][4], q1[T == kF32 ? 1 : NB][4], q2[T == kBF16 ? NB : 1][4];
    float qf[T == kF32 ? kOwn : 1][4];
    int qe;          // scores: times 2^qe
    float m, l;      // of column i: maximum, this lane's sum of weights
    f32x4 acc[kOwn]; // of column i: values (4g + r) * kOwn + e in [e][r]
    // a tile on its way
    uint32_t kw[2][T == kF32 ? kOwn : NB][T == kQ8_0 ? 2 : 4];
    static constexpr int kWords = T == kF32 ? kOwn : T == kQ8_0 ? (NB + 1) / 2 : NB;
    uint32_t vw[8][kWords];
    uint32_t ks[2][T == kQ8_0 ? 2 * NB : 1], vs[8];

    // The column's query: loaded, then (with the first keys on their way) made operands.
    float raw[T == kF32 ? kOwn : NB][T == kF32 ? 4 : 8];
    __device__ __forceinline__ void load_q(const float* q, bool some) {
        const uint32_t g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int c = 0; c < (T == kF32 ? kOwn : NB); ++c) {
#pragma unroll
            for (int j = 0; j < (T == kF32 ? 4 : 8); ++j) raw[c][j] = 0.0f;
            if (some) words<float, (T == kF32 ? 4 : 8), 4>(q + (T == kF32 ? 16 * c + 4 * g : 32 * c + 8 * g), raw[c]);
        }
    }
    __device__ __forceinline__ void start(float scale) {
        const float f = scale * 1.44269504088896340736f;  // exp(x) = 2^(x log2 e)
        m = -INFINITY, l = 0.0f, qe = 0;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) acc[e] = f32x4{0, 0, 0, 0};
        if constexpr (T == kF32) {
#pragma unroll
            for (int c = 0; c < kOwn; ++c)
#pragma unroll
                for (int j = 0; j < 4; ++j) qf[c][j] = raw[c][j] * f;
        } else {
            float top = 0.0f;
#pragma unroll
            for (int c = 0; c < NB; ++c)
#pragma unroll
                for (int j = 0; j < 8; ++j) raw[c][j] *= f, top = fmaxf(top, fabsf(raw[c][j]));
            if constexpr (T != kBF16) {  // the largest to 2^13 .. 2^14
                top = column_max(top);
                const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) : 0;
                qe = e - 14;
#pragma unroll
                for (int c = 0; c < NB; ++c)
#pragma unroll
                    for (int j = 0; j < 8; ++j) raw[c][j] = __builtin_amdgcn_ldexpf(raw[c][j], -qe);
            }
#pragma unroll
            for (int c = 0; c < NB; ++c) {
                if constexpr (T == kBF16) split_bf16(raw[c], q0[c], q1[c], q2[c]);
                else split_f16(raw[c], q0[c], q1[c]);
            }
        }
    }

    // Keys of the 16 tokens from place `row` of a plane on; half h.
    __device__ __forceinline__ void load_k(int h, const uint8_t* plane, uint32_t row, uint32_t log_page) {
        const uint32_t i = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
        const uint8_t* p = plane + (row + i) * (uint32_t)kv_row<T>(kDim);
        if constexpr (T == kQ8_0) {
#pragma unroll
            for (int c = 0; c < NB; ++c) words<uint32_t, 2, 8>(p + 32 * c + 8 * g, kw[h][c]);
            words<uint32_t, 2 * NB, pow2_of(8 * NB) < 16 ? pow2_of(8 * NB) : 16>(
                plane + ((uint32_t)kDim << log_page) + (row + 4 * g) * (2 * NB), ks[h]);
        } else {
#pragma unroll
            for (int c = 0; c < (T == kF32 ? kOwn : NB); ++c) words<uint32_t, 4, 16>(p + 64 * c + 16 * g, kw[h][c]);
        }
    }
    __device__ __forceinline__ void load_v(int h, const uint8_t* plane, uint32_t row, uint32_t log_page) {
        const uint32_t i = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t at = row + 4 * g + j;
            const uint8_t* p = plane + at * (uint32_t)kv_row<T>(kDim);
            if constexpr (T == kQ8_0) {
                if constexpr (NB % 2 == 0) {
                    words<uint32_t, kWords, pow2_of(2 * NB)>(p + i * kOwn, vw[4 * h + j]);
                } else {
                    uint16_t t[NB];
                    words<uint16_t, NB, 2>(p + i * kOwn, t);
#pragma unroll
                    for (int k = 0; k < kWords; ++k) vw[4 * h + j][k] = t[2 * k] | (2 * k + 1 < NB ? (uint32_t)t[(2 * k + 1) % NB] << 16 : 0);
                }
                // the scale of the lane's first value, and that of its last
                const uint8_t* s = plane + ((uint32_t)kDim << log_page) + at * (2 * NB);
                const uint32_t b = i * kOwn / 32, c = (i * kOwn + kOwn - 1) / 32;
                vs[4 * h + j] = *(const uint16_t*)(s + 2 * b);
                if constexpr (32 % kOwn != 0) vs[4 * h + j] |= (uint32_t)*(const uint16_t*)(s + 2 * c) << 16;
            } else {
                words<uint32_t, kWords, pow2_of(4 * kWords) < 16 ? pow2_of(4 * kWords) : 16>(p + i * (4 * kWords), vw[4 * h + j]);
            }
        }
    }

    // Scores of the loaded keys: tokens 4g + r of the halves for column i, to base 2.
    __device__ __forceinline__ void scores(float (&s)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 d = {0, 0, 0, 0};
            if constexpr (T == kF32) {
#pragma unroll
                for (int c = 0; c < kOwn; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[h][c][j]), qf[c][j], d, 0, 0, 0);
            } else if constexpr (T == kQ8_0) {
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    uint32_t a[4];  // levels as f16: 1024 + (level + 128), less 1152
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t w = kw[h][c][k / 2] ^ 0x80808080u;
                        const uint32_t u = __builtin_amdgcn_perm(0x64646464u, w, k % 2 ? 0x04030402u : 0x04010400u);
                        a[k] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, u) - (_Float16)1152.0f);
                    }
                    const f32x4 z = mma_f16(a, q1[c], mma_f16(a, q0[c], f32x4{0, 0, 0, 0}));
#pragma unroll
                    for (int r = 0; r < 4; ++r) {  // the scale of token 4g + r, block c
                        const uint32_t w = ks[h][(r * NB + c) / 2];
                        d[r] = __builtin_fmaf(half_to_float((r * NB + c) % 2 ? w >> 16 : w), z[r], d[r]);
                    }
                }
            } else {
#pragma unroll
                for (int c = 0; c < NB; ++c) {
                    if constexpr (T == kF16) d = mma_f16(kw[h][c], q1[c], mma_f16(kw[h][c], q0[c], d));
                    else d = mma_bf16(kw[h][c], q2[c], mma_bf16(kw[h][c], q1[c], mma_bf16(kw[h][c], q0[c], d)));
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * h + r] = T == kF16 || T == kQ8_0 ? __builtin_amdgcn_ldexpf(d[r], qe) : d[r];
        }
    }

    // Weights of the scores; `all`: every token counts, else those of `seen` (bit per token).
    __device__ __forceinline__ void weights(float (&s)[8], bool all, uint32_t seen) {
        if (!all) {
#pragma unroll
            for (int t = 0; t < 8; ++t) s[t] = (seen >> t) & 1 ? s[t] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int t = 1; t < 8; ++t) top = fmaxf(top, s[t]);
        if (__ballot(top > m)) {  // (rare after the first tiles)
            const float next = fmaxf(m, column_max(top));
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - next);
            m = next, l *= f;
#pragma unroll
            for (int e = 0; e < kOwn; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[e][r] *= f;
        }
        const float base = fmaxf(m, -3.402823466e38f);  // (a column that has no token yet: -inf is less)
#pragma unroll
        for (int t = 0; t < 8; ++t) s[t] = __builtin_amdgcn_exp2f(s[t] - base) * kTop;
        l += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
    }

    // Values of tokens that no column sees may be anything: they become 0.
    __device__ __forceinline__ void drop(uint32_t seen) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            if ((seen >> t) & 1) continue;
#pragma unroll
            for (int k = 0; k < kWords; ++k) vw[t][k] = 0;
            vs[t] = 0;
        }
    }

    // The tokens (bits) of which this lane holds a value that is not finite.
    __device__ __forceinline__ uint32_t not_finite() const {
        uint32_t off = 0;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            constexpr uint32_t e = T == kF32 ? 0x7f800000u : T == kBF16 ? 0x7f80u : 0x7c00u;
            bool some = false;
            if constexpr (T == kQ8_0) {
                some = (vs[t] & e) == e || (vs[t] & e << 16) == e << 16;
            } else {
#pragma unroll
                for (int k = 0; k < kWords; ++k) {
                    some |= (vw[t][k] & e) == e;
                    if constexpr (T != kF32) some |= (vw[t][k] & e << 16) == e << 16;
                }
            }
            off |= (uint32_t)some << t;
        }
        return off;
    }

    __device__ __forceinline__ void products(const float (&p)[8]) {
        if constexpr (k16) {
            uint32_t p0[4], p1[4], p2[4];
            if constexpr (T == kF16) split_f16(p, p0, p1);
            else split_bf16(p, p0, p1, p2);
#pragma unroll
            for (int e = 0; e < kOwn; ++e) {
                uint32_t a[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    a[k] = __builtin_amdgcn_perm(vw[2 * k + 1][e / 2], vw[2 * k][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
                if constexpr (T == kF16) acc[e] = mma_f16(a, p1, mma_f16(a, p0, acc[e]));
                else acc[e] = mma_bf16(a, p2, mma_bf16(a, p1, mma_bf16(a, p0, acc[e])));
            }
            return;
        }
        const uint32_t i = threadIdx.x & 15;
        // whether value e has the scale of the lane's first value
        auto same = [&](int e) { return 32 % kOwn == 0 || (i * kOwn + e) / 32 == i * kOwn / 32; };
        if constexpr (T == kQ8_0) {
            uint32_t top = 0;  // exponents and signs as they are: a scale is not negative
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const uint32_t x = vs[t] & 0xffffu, y = vs[t] >> 16;
                top = x > top ? x : top;
                if (32 % kOwn != 0) top = y > top ? y : top;
            }
            if (!__ballot(top > 0x5fffu)) {  // f16 511.75
                uint32_t p0[4], p1[4], d0[4], d1[4];
                split_f16(p, p0, p1);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    d0[k] = __builtin_amdgcn_perm(vs[2 * k + 1], vs[2 * k], 0x05040100u);
                    d1[k] = 32 % kOwn != 0 ? __builtin_amdgcn_perm(vs[2 * k + 1], vs[2 * k], 0x07060302u) : 0;
                }
#pragma unroll
                for (int e = 0; e < kOwn; ++e) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t b = __builtin_amdgcn_perm(vw[2 * k + 1][e / 4], vw[2 * k][e / 4], 0x0c040c00u + (e % 4) * 0x10001u);
                        const f16x2 q = __builtin_bit_cast(f16x2, b ^ 0x64806480u) - (_Float16)1152.0f;
                        const f16x2 d = __builtin_bit_cast(f16x2, same(e) ? d0[k] : d1[k]);
                        const f16x2 v = q * d;
                        hi[k] = __builtin_bit_cast(uint32_t, v);
                        lo[k] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(q, d, -v));
                    }
                    acc[e] = mma_f16(lo, p0, mma_f16(hi, p1, mma_f16(hi, p0, acc[e])));
                }
                return;
            }
        }
        {
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                const float s0 = half_to_float(vs[t]), s1 = half_to_float(vs[t] >> 16);
#pragma unroll
                for (int e = 0; e < kOwn; ++e) {
                    float v;
                    if constexpr (T == kF32) {
                        v = __uint_as_float(vw[t][e]);
                    } else {
                        v = (float)(int8_t)(vw[t][e / 4] >> (8 * (e % 4))) * (same(e) ? s0 : s1);
                    }
                    acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[t], acc[e], 0, 0, 0);
                }
            }
        }
    }
};

__device__ __forceinline__ void attn_put(float* to, float x, float y) {
    const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
    const unsigned long long old =
        __hip_atomic_exchange((unsigned long long*)to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    asm volatile("" ::"v"(old) : "memory");
}
__device__ __forceinline__ float2 attn_get(const float* from) {
    const unsigned long long v =
        __hip_atomic_load((const unsigned long long*)from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return make_float2(__uint_as_float((uint32_t)v), __uint_as_float((uint32_t)(v >> 32)));
}

// The tokens of all rows, in tiles of 128 row after row, are dealt evenly: slot j of a KV head (and of
// 16 of its query heads) takes `share` tiles from j * share on, whatever rows they are of.  The slots of
// all heads fill the CUs once.  A slot goes through the segments that it has of rows; four waves take 32 tokens
// of every tile, and join in LDS.  A row that lies in one slot is written by it; of others each slot puts its part where
// every workgroup can read it, and the last to arrive joins the parts in order (published as the
// router's logits are: an exchange is performed at the device's coherent level when it returns).
// So the order in which a row is added up follows from the call's rows alone, and a row whose tokens lie in one tile (an
// aligned 128 of the positions) is added up as if it were alone.
//
// Rows one behind the other of one request at one position after the other (a prompt's tokens, drafted ones) go
// together where their heads of a KV head fit a tile's 16 columns: `pack` rows at most read their tokens once.
// They differ in the first and last tokens only, which each column masks for itself; a value there that is no finite number
// is taken out and makes the columns that see it none.  With 4 query heads of 128 a KV head, f16: a prompt of 4000
// tokens 2500 us apart, 765 together; five drafted rows of each of 32 requests up to 8192 158 and 80.  Not where the
// rows apart have no more tiles than there are slots: five rows of 1000 tokens 10 us apart, on CUs of their own, 16
// together.
//
// Two workgroups a CU (registers): one loads while the other is in its prologue or joins (32 rows of 4096 tokens, 8
// KV heads of 128 in f16: one a CU 194 us, two 97).  Rows cut at multiples of 256 tokens instead of dealt: ragged
// rows (32 up to 8192) 53 us, dealt 42.
//
// Bound: HBM where there is enough to read: one row of 131072 tokens (bf16) 102 us, 5.3 TB/s; 32 rows of 4096 f16
// 96 us, 5.6; f32 184, 5.8; Q8_0 61, 4.6 (VALU issues during half of its cycles).  Small calls: six latencies
// one after another (positions, pages, keys, then parts put, counted and read): 100 tokens 6.4 us, 1000 8.6,
// 16000 21.
//
// The rows' tiles are counted by every workgroup: to 64 rows a lane each, else in LDS.
template <uint32_t T, int NB>
__global__ __launch_bounds__(256, NB <= attn_wide(T) ? 2 : 1) void kv_attention_kernel(AttnArgs a) {
    constexpr uint32_t kDim = 32 * NB, kLine = kDim + 2, kV = (kDim + 127) / 128;
    __shared__ uint32_t start[kAttnRows + 1], sums[4], mosts[4], begins[4], runs[4];
    __shared__ int32_t firsts[kAttnRows], lasts[kAttnRows], of[kAttnRows];
    __shared__ uint8_t size[kAttnRows];
    __shared__ __align__(16) float part[4][16][kLine];  // of a wave and column: values
    __shared__ float wave_m[4][16], wave_l[4][16];
    __shared__ uint32_t last_one;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, g = lane >> 4;
    const uint32_t group = a.heads / a.c.kv_heads, tiles = (group + 15) / 16, per = a.c.kv_heads * tiles;
    const uint32_t pack = a.pack, line = (group < 16 ? pack * group : 16) * (kDim + 2);  // floats of a part

    // a row's request (-1: left alone), first and last token
    auto span = [&](uint32_t row, int32_t& request, int32_t& first, int32_t& last) {
        request = a.requests ? a.requests[row] : (int32_t)row, last = a.positions[row];
        first = a.window && (uint32_t)last + 1 > a.window ? (int32_t)((uint32_t)last + 1 - a.window) : 0;
        if (request >= 0 && (uint32_t)request < a.table_rows && last >= -1 && last < (int64_t)a.width << a.c.log_page) return;
        if (request != -1) report_error(a.err_word, bounds_key(a.row0 + row));
        request = -1;
    };
    auto follows = [](int32_t request, int32_t last, int32_t request0, int32_t last0) {  // the row before
        return request >= 0 && request == request0 && last0 >= 0 && last - 1 == last0;
    };
    auto tiles_of = [](int32_t first, int32_t last) { return last < 0 ? 1u : ((uint32_t)last >> 7) - ((uint32_t)first >> 7) + 1; };
    const bool few = a.rows <= 64;
    // few: of row `lane`; the first of those that go together has their number and their tiles, the others none
    int32_t my_request = -1, my_first = 0, my_last = -1;
    uint32_t my_rows = 1, my_start = 0, my_tiles = 0, total, longest;
    if (few) {
        if (lane < a.rows) span(lane, my_request, my_first, my_last);
        my_tiles = my_request >= 0 ? tiles_of(my_first, my_last) : 0;
        uint32_t sum = wave_scan_u32(my_tiles);
        total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        const bool on = follows(my_request, my_last, __shfl_up(my_request, 1, 64), __shfl_up(my_last, 1, 64)) && lane > 0;
        const unsigned long long breaks = __ballot(!on);
        if (pack > 1 && total > a.slots && ~breaks) {
            const uint32_t run = 63 - (uint32_t)__builtin_clzll(breaks & ((2ull << lane) - 1));
            const unsigned long long heads = __ballot((lane - run) % pack == 0), after = lane < 63 ? heads >> (lane + 1) : 0;
            my_rows = (heads >> lane) & 1 ? (after ? (uint32_t)__builtin_ctzll(after) + 1 : 64 - lane) : 0;
            my_tiles = my_request >= 0 && my_rows ? tiles_of(my_first, my_last + (int32_t)(my_rows - 1)) : 0;
            sum = wave_scan_u32(my_tiles);
            total = (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
        }
        my_start = sum - my_tiles;
        longest = wave_max_u32(my_tiles);
    } else {
        constexpr uint32_t kMine = kAttnRows / 256;
        uint32_t n[kMine], begin = 0, sum, mine;  // begin: the last of the thread's rows that does not follow the one before
        bool on[kMine], any = false;
        int32_t request0 = -1, last0 = -1;
        const uint32_t row0 = tid * kMine;
        if (row0 > 0 && row0 < a.rows) request0 = a.requests ? a.requests[row0 - 1] : -1, last0 = a.positions[row0 - 1];
#pragma unroll
        for (uint32_t k = 0; k < kMine; ++k) {
            const uint32_t row = row0 + k;
            n[k] = 0, on[k] = false;
            if (row >= a.rows) continue;
            int32_t request, first, last;
            span(row, request, first, last);
            on[k] = follows(request, last, request0, last0);
            request0 = request, last0 = last;
            firsts[row] = first, lasts[row] = last, of[row] = request, size[row] = 1;
            n[k] = request >= 0 ? tiles_of(first, last) : 0;
            begin = on[k] ? begin : row;
            any |= on[k];
        }
        auto scan = [&] {  // of the rows' tiles
            mine = 0;
            uint32_t most = 0;
#pragma unroll
            for (uint32_t k = 0; k < kMine; ++k) mine += n[k], most = n[k] > most ? n[k] : most;
            sum = wave_scan_u32(mine);
            most = wave_max_u32(most);
            if (lane == 63) sums[wave] = sum, mosts[wave] = most;
        };
        scan();
        const bool some_on = __ballot(any) != 0;
        if (lane == 63) runs[wave] = some_on;
        __syncthreads();
        any = (runs[0] | runs[1] | runs[2] | runs[3]) != 0;
        total = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (pack > 1 && total > a.slots && any) {
            // the beginning of the row's run, of all threads before this one
            uint32_t upto = begin;
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t o = __shfl_up(upto, m, 64);
                upto = (int)lane >= m && o > upto ? o : upto;
            }
            if (lane == 63) begins[wave] = upto;
            upto = __shfl_up(upto, 1, 64);
            upto = lane ? upto : 0;
            __syncthreads();
            for (uint32_t w = 0; w < wave; ++w) upto = begins[w] > upto ? begins[w] : upto;
#pragma unroll
            for (uint32_t k = 0; k < kMine; ++k) {
                const uint32_t row = row0 + k;
                if (row >= a.rows) continue;
                upto = on[k] ? upto : row;
                const uint32_t at = (row - upto) % pack;
                if (at) size[row] = 0;
                // (the last of those that go together tells the first)
                const bool end = row + 1 == a.rows || at + 1 == pack || !follows(of[row + 1], lasts[row + 1], of[row], lasts[row]);
                if (at && end) size[row - at] = (uint8_t)(at + 1);
            }
            __syncthreads();
#pragma unroll
            for (uint32_t k = 0; k < kMine; ++k) {
                const uint32_t row = row0 + k;
                if (row >= a.rows) continue;
                n[k] = of[row] >= 0 && size[row] ? tiles_of(firsts[row], lasts[row] + (size[row] - 1)) : 0;
            }
            scan();
            __syncthreads();
        }
        sum -= mine;
        longest = 0;
        for (uint32_t w = 0; w < 4; ++w) longest = mosts[w] > longest ? mosts[w] : longest;
        for (uint32_t w = 0; w < wave; ++w) sum += sums[w];
#pragma unroll
        for (uint32_t k = 0; k < kMine; ++k) {
            const uint32_t row = row0 + k;
            if (row <= a.rows) start[row] = sum;
            sum += n[k];
            if (row + 1 == kAttnRows) start[kAttnRows] = sum;
        }
        __syncthreads();
        total = start[a.rows];
    }
    // A row has kAttnParts parts at most, which one wave's lanes join: of n tiles, in twos or more, wherever it begins in its
    // first slot, at most (n - 2) / share + 2.  And 32 parts of one tile are joined in the time that 16 of two take
    // more: 4000 tokens of two KV heads of 64 13.4 us and 11.9, 16 rows of 4096 with one of 128 18.7 and 15.6.
    const uint32_t least = total / a.slots + (total % a.slots != 0);
    const uint32_t joined = longest > 16 ? (longest - 2) / (kAttnParts - 1) + 1 : 1;
    const uint32_t row_least = longest > 16 && joined < 2 ? 2 : joined;
    const uint32_t share = least < row_least ? row_least : least;
    const uint32_t slot = blockIdx.x / per, hc = blockIdx.x - slot * per, kvh = hc / tiles;
    const uint32_t wide = group - 16 * (hc - kvh * tiles) < 16 ? group - 16 * (hc - kvh * tiles) : 16;  // heads of a row
    const uint32_t my_row = i / wide;  // column i's among those that go together
    const uint32_t head0 = kvh * group + 16 * (hc - kvh * tiles);
    const uint64_t plane = kvh * kv_plane<T>(kDim, a.c.log_page);
    const uint32_t mask = (1u << a.c.log_page) - 1;
    const uint64_t end64 = (uint64_t)(slot + 1) * share;
    const uint32_t end = end64 < total ? (uint32_t)end64 : total;

    uint32_t next;
    for (uint64_t tile = (uint64_t)slot * share; tile < end; tile = next) {
        uint32_t row, row0, row1, rows;
        int32_t request, first, last;  // last: the first row's
        if (few) {
            row = 63 - (uint32_t)__builtin_clzll(__ballot(my_tiles > 0 && my_start <= tile));
            row0 = (uint32_t)__builtin_amdgcn_readlane((int)my_start, (int)row);
            row1 = row0 + (uint32_t)__builtin_amdgcn_readlane((int)my_tiles, (int)row);
            request = __builtin_amdgcn_readlane(my_request, (int)row);
            first = __builtin_amdgcn_readlane(my_first, (int)row), last = __builtin_amdgcn_readlane(my_last, (int)row);
            rows = (uint32_t)__builtin_amdgcn_readlane((int)my_rows, (int)row);
        } else {
            row = (uint32_t)__builtin_amdgcn_readfirstlane((int)segment_of(start, a.rows, (uint32_t)tile));
            row0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)start[row]);
            row1 = (uint32_t)__builtin_amdgcn_readfirstlane((int)start[row + 1]);
            request = __builtin_amdgcn_readfirstlane(of[row]);
            first = __builtin_amdgcn_readfirstlane(firsts[row]), last = __builtin_amdgcn_readfirstlane(lasts[row]);
            rows = (uint32_t)__builtin_amdgcn_readfirstlane((int)size[row]);
        }
        next = row1 < end ? row1 : end;
        const uint32_t slot0 = row0 / share, parts = (row1 - 1) / share - slot0 + 1;
        const uint32_t cols = rows * wide;
        // of the segment's tokens, t0 to before t1 (from a tile's beginning on), column i sees s0 to before s1, all
        // columns see a0 to before a1 (positions are below 2^31)
        const uint32_t from = (((uint32_t)first >> 7) + (uint32_t)(tile - row0)) << 7, to = from + ((uint32_t)(next - tile) << 7);
        const uint32_t seen0 = (uint32_t)last + 1;  // that the first row sees
        auto first_of = [&](uint32_t k) { return a.window && seen0 + k > a.window ? seen0 + k - a.window : 0; };  // row k
        const uint32_t t0 = from > (uint32_t)first ? from : (uint32_t)first, t1 = to < last + rows ? to : last + rows;
        const uint32_t mine_of = my_row < rows ? my_row : rows - 1;  // (columns behind the last: as the last row's)
        const uint32_t fm = first_of(mine_of), s0 = t0 > fm ? t0 : fm, s1 = t1 < seen0 + mine_of ? t1 : seen0 + mine_of;
        const uint32_t fa = first_of(rows - 1), a0 = t0 > fa ? t0 : fa, a1 = t1 < seen0 ? t1 : seen0;

        AttnWave<T, NB> w;
        const int32_t* table = a.tables + (uint64_t)request * a.width;
        bool lost = false;
        int32_t id = 0;
        uint32_t c0 = from;
        // lane k: the page of the sixteen tokens from c0 + 16 k on
        auto pages = [&](uint32_t c0) {
            const uint32_t at = c0 + 16 * lane;
            id = 0;
            if (at < t1 && at + 16 > t0) id = table[at >> a.c.log_page];
        };
        auto check = [&] {
            const bool off = id < 0 || (uint64_t)id >= a.c.pages;
            for (unsigned long long m = __ballot(off); m; m &= m - 1) {  // (a column that sees none of its tokens keeps on)
                const uint32_t at = c0 + 16 * (uint32_t)__builtin_ctzll(m);
                lost |= at < s1 && at + 16 > s0;
            }
            if (off) id = 0;
        };
        auto page = [&](uint32_t t) { return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(id, (int)((t - c0) >> 4)); };
        auto load_k = [&](uint32_t t) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                w.load_k(h, a.c.k + page(t + 16 * h) * a.c.k_stride + plane, (t + 16 * h) & mask, a.c.log_page);
        };
        auto load_v = [&](uint32_t t) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                w.load_v(h, a.c.v + page(t + 16 * h) * a.c.v_stride + plane, (t + 16 * h) & mask, a.c.log_page);
        };
        pages(c0);
        w.load_q(a.q + (row + my_row) * a.q_stride + (uint64_t)(head0 + i - my_row * wide) * kDim, i < cols);
        check();
        if (c0 + 32 * wave < t1) load_k(c0 + 32 * wave), load_v(c0 + 32 * wave);
        w.start(a.scale);
        for (;;) {
            const uint32_t c1 = c0 + 1024 < t1 ? c0 + 1024 : t1;
            for (uint32_t t = c0 + 32 * wave; t < c1; t += 128) {
                const bool all = t >= a0 && t + 32 <= a1, more = t + 128 < c1;
                uint32_t seen = 0;
                if (!all) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint32_t tok = t + 16 * (k / 4) + 4 * g + k % 4;
                        seen |= (uint32_t)(tok >= s0 && tok < s1) << k;
                    }
                }
                float s[8];
                w.scores(s);
                if (more) load_k(t + 128);
                w.weights(s, all, seen);
                if (!all) {
                    uint32_t some = seen;
                    if (rows > 1) {  // the tokens that some column sees and whose values all are finite
                        uint32_t off = w.not_finite();
                        some = 0;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const uint32_t tok = t + 16 * (k / 4) + 4 * g + k % 4;
                            some |= (uint32_t)(tok >= t0 && tok < t1) << k;
                        }
                        off |= __shfl_xor(off, 1, 64), off |= __shfl_xor(off, 2, 64);
                        off |= __shfl_xor(off, 4, 64), off |= __shfl_xor(off, 8, 64);
                        if (off & seen) w.l = NAN;
                        some &= ~off;
                    }
                    w.drop(some);
                }
                w.products(s);
                if (more) load_v(t + 128);
            }
            if (c0 + 1024 >= t1) break;
            c0 += 1024;
            pages(c0);
            check();
            if (c0 + 32 * wave < t1) load_k(c0 + 32 * wave), load_v(c0 + 32 * wave);
        }
        if (lost && i < cols) {  // (every segment finds its own; what is joined is then no number)
            w.l = NAN;
            report_error(a.err_word, bounds_key(a.row0 + row + my_row));
        }

        // the waves join
        w.l = column_sum(w.l);
        if (g == 0) wave_m[wave][i] = w.m, wave_l[wave][i] = w.l;
        __syncthreads();
        const float top = fmaxf(fmaxf(wave_m[0][i], wave_m[1][i]), fmaxf(wave_m[2][i], wave_m[3][i]));
        const float f = w.m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(w.m - top);
        if (i < cols) {
#pragma unroll
            for (int e = 0; e < 2 * NB; ++e)
#pragma unroll
                for (int r = 0; r < 4; ++r) part[wave][i][(4 * g + r) * (2 * NB) + e] = w.acc[e][r] * f;
        }
        __syncthreads();
        auto write = [&](uint32_t c, float (&y)[kV][2], float sum) {  // column c's values 2 lane + 128 k and the next
            bool off = false;
#pragma unroll
            for (uint32_t k = 0; k < kV; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    y[k][j] = last < 0 ? 0.0f : y[k][j] / sum;
                    off |= 2 * lane + 128 * k < kDim && !finite(y[k][j]);
                }
            if (__ballot(off)) {
                if (lane == 0) report_error(a.err_word, model_key(a.row0 + row + c / wide, kStAttnOut, 0));
                return;
            }
            float* out = a.out + (row + c / wide) * a.out_stride + (uint64_t)(head0 + c % wide) * kDim;
#pragma unroll
            for (uint32_t k = 0; k < kV; ++k) {
                const uint32_t d = 2 * lane + 128 * k;
                if (d < kDim) out[d] = y[k][0], out[d + 1] = y[k][1];
            }
        };
        // a wave takes every fourth column
        auto scratch = [&](uint32_t k) {  // part k of the row; a slot ends one row that goes on and begins one
            return a.scratch + (((uint64_t)hc * a.slots + slot0 + k) * 2 + (k == 0)) * line;
        };
        float* mine = scratch(slot - slot0);
        for (uint32_t c = wave; c < cols; c += 4) {
            const float ct = fmaxf(fmaxf(wave_m[0][c], wave_m[1][c]), fmaxf(wave_m[2][c], wave_m[3][c]));
            float sum = 0.0f, y[kV][2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float l = wave_l[k][c];
                sum += l == 0.0f ? 0.0f : l * __builtin_amdgcn_exp2f(wave_m[k][c] - ct);  // (0: without tokens)
            }
#pragma unroll
            for (uint32_t k = 0; k < kV; ++k) {
                const uint32_t d = 2 * lane + 128 * k;
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    y[k][j] = d < kDim ? (part[0][c][d + j] + part[1][c][d + j]) + (part[2][c][d + j] + part[3][c][d + j]) : 0.0f;
            }
            if (parts == 1) {
                write(c, y, sum);
                continue;
            }
#pragma unroll
            for (uint32_t k = 0; k < kV; ++k)
                if (2 * lane + 128 * k < kDim) attn_put(mine + c * (kDim + 2) + 2 * lane + 128 * k, y[k][0], y[k][1]);
            if (lane == 0) attn_put(mine + c * (kDim + 2) + kDim, ct, sum);
        }
        __syncthreads();
        if (parts == 1) continue;
        if (tid == 0) {
            uint32_t* count = a.count + (uint64_t)hc * a.slots + slot0;
            const uint32_t old = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            last_one = old == parts - 1;
            if (last_one) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
        __syncthreads();
        if (!last_one) continue;
        constexpr uint32_t kBatch = 8 / kV;  // parts on their way
        for (uint32_t c = wave; c < cols; c += 4) {
            const uint32_t at = c * (kDim + 2);
            float2 ml[2];  // of parts `lane` and lane + 64
#pragma unroll
            for (uint32_t k = 0; k < 2; ++k)
                ml[k] = lane + 64 * k < parts ? attn_get(scratch(lane + 64 * k) + at + kDim) : make_float2(-INFINITY, 0.0f);
            float fs[2], sum, y[kV][2] = {};
            for (uint32_t k0 = 0; k0 < parts; k0 += kBatch) {
                float2 x[kBatch][kV];
#pragma unroll
                for (uint32_t k = 0; k < kBatch; ++k)
#pragma unroll
                    for (uint32_t v = 0; v < kV; ++v)
                        x[k][v] = k0 + k < parts && 2 * lane + 128 * v < kDim ? attn_get(scratch(k0 + k) + at + 2 * lane + 128 * v)
                                                                              : make_float2(0.0f, 0.0f);
                if (k0 == 0) {
                    const float ct = wave_max_dpp(fmaxf(ml[0].x, ml[1].x));
#pragma unroll
                    for (int k = 0; k < 2; ++k) fs[k] = __builtin_amdgcn_exp2f(ml[k].x - ct);
                    sum = wave_sum(ml[0].y * fs[0] + ml[1].y * fs[1]);
                }
#pragma unroll
                for (uint32_t k = 0; k < kBatch; ++k) {
                    if (k0 + k >= parts) continue;
                    const float fk = readlane_f(k0 + k < 64 ? fs[0] : fs[1], (int)((k0 + k) & 63));
#pragma unroll
                    for (uint32_t v = 0; v < kV; ++v) {
                        y[v][0] = __builtin_fmaf(x[k][v].x, fk, y[v][0]);
                        y[v][1] = __builtin_fmaf(x[k][v].y, fk, y[v][1]);
                    }
                }
            }
            write(c, y, sum);
        }
        __syncthreads();
    }
}

// Slots of a KV head (and 16 of its query heads); the rows of a launch, whose tiles are counted in 32 bits.
static uint32_t attn_slots(const AttnArgs& a) {
    const uint32_t per = a.c.kv_heads * ((a.heads / a.c.kv_heads + 15) / 16);
    const uint32_t wide = attn_wide(a.c.type), n = (a.c.dim / 32 <= wide ? 2u : 1u) * (uint32_t)device_cus() / per;
    return n < 1 ? 1 : n;
}
static uint32_t attn_rows(const AttnArgs& a) {
    const uint64_t tokens = (uint64_t)a.width << a.c.log_page, tiles = (tokens < 1ull << 31 ? tokens : 1ull << 31) / 128 + 2;
    const uint64_t n = 0xffffffffull / tiles;
    return (uint32_t)(n < kAttnRows ? n : kAttnRows);
}
// Rows that go together at most: of those that fill a tile's columns.
static uint32_t attn_pack(const AttnArgs& a) {
    const uint32_t group = a.heads / a.c.kv_heads;
    return group > 8 || a.rows == 1 || !a.requests ? 1 : 16 / group;
}
size_t kv_attention_bytes(const AttnArgs& a) {
    const uint64_t group = a.heads / a.c.kv_heads, per = a.c.kv_heads * ((group + 15) / 16);
    if (attn_slots(a) == 1) return 0;  // (every row in one slot)
    return per * attn_slots(a) * 2 * (group < 16 ? attn_pack(a) * group : 16) * (a.c.dim + 2) * sizeof(float);
}
uint64_t kv_attention_counters(const AttnArgs& a) {
    return (uint64_t)a.c.kv_heads * ((a.heads / a.c.kv_heads + 15) / 16) * attn_slots(a);
}

template <uint32_t T, int NB>
static void attn_launch(const AttnArgs& a, uint32_t grid, hipStream_t s) {
    hipLaunchKernelGGL((kv_attention_kernel<T, NB>), dim3(grid), dim3(256), 0, s, a);
}
template <uint32_t T>
static hipError_t attn_dims(const AttnArgs& a, uint32_t grid, hipStream_t s) {
    switch (a.c.dim / 32) {
        case 1: attn_launch<T, 1>(a, grid, s); break;
        case 2: attn_launch<T, 2>(a, grid, s); break;
        case 3: attn_launch<T, 3>(a, grid, s); break;
        case 4: attn_launch<T, 4>(a, grid, s); break;
        case 5: attn_launch<T, 5>(a, grid, s); break;
        case 6: attn_launch<T, 6>(a, grid, s); break;
        case 7: attn_launch<T, 7>(a, grid, s); break;
        case 8: attn_launch<T, 8>(a, grid, s); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_kv_attention(AttnArgs a, hipStream_t s) {
    if (a.rows == 0 || a.rows > 65535 || a.heads == 0 || a.heads > 65535 || a.c.dim % 32 || a.c.dim > 256 ||
        a.heads % a.c.kv_heads)
        return hipErrorInvalidValue;
    a.slots = attn_slots(a);
    a.pack = attn_pack(a);
    const uint32_t rows = a.rows, most = attn_rows(a), grid = (uint32_t)kv_attention_counters(a);
    const AttnArgs all = a;
    for (uint32_t r = 0; r < rows; r += most) {  // (the parts and counters are the same memory)
        a.row0 = r;
        a.rows = rows - r < most ? rows - r : most;
        a.q = all.q + r * a.q_stride, a.out = all.out + r * a.out_stride, a.positions = all.positions + r;
        if (all.requests) a.requests = all.requests + r;
        else a.tables = all.tables + (uint64_t)r * a.width, a.table_rows = all.table_rows - r;  // (row t is request t)
        hipError_t e;
        switch (a.c.type) {
            case kF32: e = attn_dims<kF32>(a, grid, s); break;
            case kF16: e = attn_dims<kF16>(a, grid, s); break;
            case kBF16: e = attn_dims<kBF16>(a, grid, s); break;
            case kQ8_0: e = attn_dims<kQ8_0>(a, grid, s); break;
            default: return hipErrorInvalidValue;
        }
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

// ---------------------------------------------------------------------------
// The beams' tables
// ---------------------------------------------------------------------------

// A group's beams after a choice: beam b goes on from parents[b] (-1: from itself).
// Whole pages are shared: their columns of the tables are the parent's.  The page that
// is being filled is each beam's own: its first tokens are copied, in every tensor.
// A thread takes one column, or one piece at one place of all beams' pages: it has
// loaded all before it stores any, so the beams may change places among themselves.
//
// Bound: the stores: eight groups of eight beams, 16 tensors of 8 heads of 57 rows of 256 bytes, 32 us (with branches
// between the loads the pieces went through scratch memory: 61); one group of four in two layers 3.8 us, two
// latencies and a launch.
//
// grid: runs of pieces (or of columns), groups, tensors (the tables first).
// (lane b holds beam b's page and that of its parent; lanes behind the last beam the first beam's.  A beam
// that stays is loaded too: it is some other's parent in most cases, and no branch lies between the loads)
template <int MB, class V>
__device__ __forceinline__ void reorder_piece(uint8_t* at, uint64_t stride, int32_t page, int32_t source, uint32_t moved) {
    V v[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) v[b] = *(const V*)(at + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(source, b) * stride);
#pragma unroll
    for (int b = 0; b < MB; ++b)
        if ((moved >> b) & 1) *(V*)(at + (uint64_t)(uint32_t)__builtin_amdgcn_readlane(page, b) * stride) = v[b];
}

template <int MB>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a) {
    const uint32_t tid = threadIdx.x, lane = tid & 63, g = blockIdx.y, B = a.beams;
    const uint64_t beam0 = (uint64_t)g * B;
    // lane b of every wave: beam b
    const bool some = lane < B;
    const int32_t len0 = a.lengths[beam0], len = some ? a.lengths[beam0 + lane] : len0;
    const int32_t p = some ? a.parents[beam0 + lane] : -1;
    const uint32_t tail = (uint32_t)(len0 < 0 ? 0 : len0) >> a.log_page, rows = (uint32_t)len0 & ((1u << a.log_page) - 1);
    bool wrong = p < -1 || p >= (int32_t)B || len < 0 || len != len0 || (uint64_t)tail + (rows > 0) > a.width;
    const bool off = __ballot(wrong) != 0;
    int32_t page = 0;
    if (!off && rows && some) {
        page = a.tables[(beam0 + lane) * a.width + tail];
        wrong = page < 0 || (uint64_t)page >= a.pages;
    }
    if (__ballot(wrong)) {  // (every wave of the group's workgroups finds the same)
        if (wrong) report_error(a.err_word, bounds_key(beam0 + lane));
        return;
    }
    const int32_t parent = p == -1 ? (int32_t)lane : p;
    const uint32_t moved = (uint32_t)__ballot(some && parent != (int32_t)lane);
    if (!moved) return;
    if (blockIdx.z == 0) {
        if (!a.last) return;  // (the tables are taken over by the last launch)
        for (uint32_t c = blockIdx.x * 256 + tid; c < tail; c += gridDim.x * 256) {
            int32_t v[MB] = {};
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if ((moved >> b) & 1) v[b] = a.tables[(beam0 + (uint32_t)__builtin_amdgcn_readlane(parent, b)) * a.width + c];
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if ((moved >> b) & 1) a.tables[(beam0 + b) * a.width + c] = v[b];
        }
        return;
    }
    if (!rows) return;
    uint8_t* base = a.tensors[blockIdx.z - 1];
    const uint64_t stride = (blockIdx.z - 1) & 1 ? a.v_stride : a.k_stride;
    const int32_t source = __shfl(page, some ? parent : 0, 64);
    // a plane's rows in use, as pieces of 16 bytes; Q8_0: and the scales' in pieces of 2
    const uint32_t plane = (a.row_bytes + a.scale_bytes) << a.log_page;
    const uint32_t pieces = rows * a.row_bytes / 16, scales = rows * a.scale_bytes / 2;
    for (uint32_t h = blockIdx.x; h < a.kv_heads * a.slices; h += gridDim.x) {
        const uint32_t head = h / a.slices, slice = h - head * a.slices;
        const uint64_t at = (uint64_t)head * plane;
#pragma unroll 1
        for (uint32_t i = slice * 256 + tid; i < pieces; i += a.slices * 256)
            reorder_piece<MB, u32x4>(base + at + 16 * i, stride, page, source, moved);
        const uint64_t after = at + ((uint64_t)a.row_bytes << a.log_page);
#pragma unroll 1
        for (uint32_t i = slice * 256 + tid; i < scales; i += a.slices * 256)
            reorder_piece<MB, uint16_t>(base + after + 2 * i, stride, page, source, moved);
    }
}

hipError_t launch_beam_reorder(ReorderArgs a, hipStream_t s) {
    if (a.groups == 0 || a.groups > 65535 || a.beams == 0 || a.beams > kReorderMaxBeams || a.n_tensors > 2 * kReorderLayers)
        return hipErrorInvalidValue;
    // a workgroup takes a head's plane, or a slice of it, so that there are some thousand of them
    const uint64_t units = (uint64_t)a.groups * a.n_tensors * a.kv_heads, most = ((a.row_bytes << a.log_page) / 16 + 255) / 256;
    a.slices = units >= 2048 ? 1 : (uint32_t)((2048 + units - 1) / units);
    if (a.slices > most) a.slices = (uint32_t)most;
    // (a launch of 2^32 threads would not run whole)
    const uint64_t x = (uint64_t)a.kv_heads * a.slices, fits = (1ull << 31) / ((uint64_t)a.groups * (1 + a.n_tensors) * 256);
    const dim3 grid((uint32_t)(x < fits ? x : fits < 1 ? 1 : fits), a.groups, 1 + a.n_tensors), block(256);
    if (a.beams <= 4) hipLaunchKernelGGL(beam_reorder_kernel<4>, grid, block, 0, s, a);
    else if (a.beams <= 8) hipLaunchKernelGGL(beam_reorder_kernel<8>, grid, block, 0, s, a);
    else if (a.beams <= 16) hipLaunchKernelGGL(beam_reorder_kernel<16>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(beam_reorder_kernel<kReorderMaxBeams>, grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace rlq
