// Rotary positions for gfx950: of every head's columns the first 2 * pairs are turned, pair i by the angle position * f_i, as
// neighbouring columns (2i, 2i + 1) or as halves (i, i + pairs):
//   a' = amplitude (a cos - b sin),   b' = amplitude (a sin + b cos).
// The columns behind them are handed on as they are.
//
// The angle. f_i comes as a share of a turn per position in 64 bits of fixed point, so that position * f_i modulo 2^64 is the share of
// a turn that is left, without any reduction and without an error of its own, where a product of floats is off by whole turns beyond 2^24. (The table's own
// error counts position times: shares made in 64-bit floating point, as the framework's are, are off by up to 2^-54 turns.) The top 32 bits are taken. The quarter of a turn next to it is taken off in whole numbers; what is left, at most an eighth of a turn, goes to
// a float (off by 2^-24 of itself) and into the series of sine and cosine, cut where the next term is below 2e-9 and 2e-10 of 1.
//
// Bound by memory: every row is read and written once. A thread has one place of a head (16 bytes; with halves the 16 bytes of both
// halves), works out its angles once and goes through the heads with them. 8,192 rows of 40 heads of 128 in bfloat16 take 36 us, 4.6 TB/s, where a
// copy of as many bytes reaches 5.2 (32 us); four heads' loads on their way at once instead of one's: 35.8 us, no more than runs differ. Where pairs, head or
// strides do not fill 16 bytes it is a column (halves) or a pair (neighbours) at a time: 8,192 rows of 40 heads of 80 with 20 columns as halves take 79 us, 1.3 TB/s. 200 rows of 18
// heads of 96 in 32 bits take 3.2 us, a launch; the call 7.1, which the host takes to make it.
#include "common.h"

#include <algorithm>

#define ROT_THREADS 256

namespace {

__device__ __forceinline__ void turn_of(int position, unsigned long long share, float amplitude, float& c, float& s) {
    const unsigned top = static_cast<unsigned>((static_cast<unsigned long long>(static_cast<long long>(position)) * share) >> 32);
    const unsigned quarter = (top + 0x20000000u) >> 30;
    const float x = static_cast<float>(static_cast<int>(top - (quarter << 30))) * 1.46291807926715968105e-9f;        // (2 pi / 2^32)
    const float z = x * x;
    const float sn = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), x);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.f);
    const bool swap = quarter & 1;
    const float cv = swap ? sn : cs, sv = swap ? cs : sn;
    c = amplitude * ((quarter + 1) & 2 ? -cv : cv);
    s = amplitude * (quarter & 2 ? -sv : sv);
}

template <typename T, int V> struct Piece;
template <> struct Piece<float, 4> {
    __device__ static void load(const float* p, float (&v)[4]) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    }
    __device__ static void store(float* p, const float (&v)[4]) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
};
template <> struct Piece<bf16_t, 8> {
    __device__ static void load(const bf16_t* p, float (&v)[8]) { load8(p, v); }
    __device__ static void store(bf16_t* p, const float (&v)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
};
template <typename T> struct Piece<T, 2> {
    __device__ static void load(const T* p, float (&v)[2]) { v[0] = to_float(p[0]); v[1] = to_float(p[1]); }
    __device__ static void store(T* p, const float (&v)[2]) { p[0] = from_float<T>(v[0]); p[1] = from_float<T>(v[1]); }
};
template <typename T> struct Piece<T, 1> {
    __device__ static void load(const T* p, float (&v)[1]) { v[0] = to_float(p[0]); }
    __device__ static void store(T* p, const float (&v)[1]) { p[0] = from_float<T>(v[0]); }
};

// V columns at a time. Places of a head: with halves, pairs / V that are turned, then those of the columns behind; otherwise head_dim / V.
template <typename T, int V, bool HALVES>
__global__ void __launch_bounds__(ROT_THREADS)
rotary_kernel(const T* x, T* out, const int* __restrict__ positions, const unsigned long long* __restrict__ turns, int tokens, int pairs, int n_heads,
              int head_dim, long long ldx, long long ldo, int places, int heads_each, float amplitude) {
    const long long item = static_cast<long long>(blockIdx.x) * ROT_THREADS + threadIdx.x;
    if (item / places >= tokens) return;
    const int t = static_cast<int>(item / places), place = static_cast<int>(item % places);
    const int position = positions[t], h0 = blockIdx.y * heads_each, h1 = min(h0 + heads_each, n_heads);
    const T* from = x + t * ldx;
    T* to = out + t * ldo;
    if constexpr (HALVES) {
        if (place < pairs / V) {
            float c[V], s[V];
#pragma unroll
            for (int e = 0; e < V; ++e) turn_of(position, turns[place * V + e], amplitude, c[e], s[e]);
            for (int h = h0; h < h1; ++h) {
                const size_t at = static_cast<size_t>(h) * head_dim + place * V;
                float a[V], b[V], u[V], v[V];
                Piece<T, V>::load(from + at, a);
                Piece<T, V>::load(from + at + pairs, b);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    u[e] = a[e] * c[e] - b[e] * s[e];
                    v[e] = a[e] * s[e] + b[e] * c[e];
                }
                Piece<T, V>::store(to + at, u);
                Piece<T, V>::store(to + at + pairs, v);
            }
            return;
        }
        const int col = 2 * pairs + (place - pairs / V) * V;
        for (int h = h0; h < h1; ++h) {
            float a[V];
            Piece<T, V>::load(from + static_cast<size_t>(h) * head_dim + col, a);
            Piece<T, V>::store(to + static_cast<size_t>(h) * head_dim + col, a);
        }
    } else {
        constexpr int P = V / 2;
        float c[P], s[P];
#pragma unroll
        for (int e = 0; e < P; ++e) {
            c[e] = 1.f; s[e] = 0.f;
            if (place * P + e < pairs) turn_of(position, turns[place * P + e], amplitude, c[e], s[e]);
        }
        for (int h = h0; h < h1; ++h) {
            const size_t at = static_cast<size_t>(h) * head_dim + place * V;
            float a[V], u[V];
            Piece<T, V>::load(from + at, a);
#pragma unroll
            for (int e = 0; e < P; ++e) {
                const bool turned = place * P + e < pairs;
                u[2 * e] = turned ? a[2 * e] * c[e] - a[2 * e + 1] * s[e] : a[2 * e];
                u[2 * e + 1] = turned ? a[2 * e] * s[e] + a[2 * e + 1] * c[e] : a[2 * e + 1];
            }
            Piece<T, V>::store(to + at, u);
        }
    }
}

template <typename T>
int launch_rotary(const T* x, long long ldx, const int* positions, const unsigned long long* turns, int tokens, int pairs, int n_heads, int head_dim,
                  int interleaved, float amplitude, T* out, long long ldo, hipStream_t stream) {
    constexpr int W = 16 / sizeof(T);
    const bool in_place = static_cast<const void*>(x) == static_cast<const void*>(out);
    const bool wide = head_dim % W == 0 && ldx % W == 0 && ldo % W == 0 && reinterpret_cast<uintptr_t>(x) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0 &&
                      (interleaved || pairs % W == 0);
    auto launch = [&](auto width_tag, auto halves_tag) {
        constexpr int V = decltype(width_tag)::value;
        constexpr bool HALVES = decltype(halves_tag)::value;
        // (in place the columns behind are there already)
        const int places = HALVES ? pairs / V + (in_place ? 0 : (head_dim - 2 * pairs) / V) : in_place ? (2 * pairs + V - 1) / V : head_dim / V;
        if (places == 0) return 0;
        const long long items = static_cast<long long>(tokens) * places, blocks = (items + ROT_THREADS - 1) / ROT_THREADS;
        if (blocks * ROT_THREADS > UINT32_MAX) return -1;             // (what one launch can have)
        const int slices = static_cast<int>(std::min<long long>(n_heads, std::max<long long>(1, 1024 / blocks)));
        const int each = (n_heads + slices - 1) / slices;
        rotary_kernel<T, V, HALVES><<<dim3(static_cast<unsigned>(blocks), (n_heads + each - 1) / each), ROT_THREADS, 0, stream>>>(
            x, out, positions, turns, tokens, pairs, n_heads, head_dim, ldx, ldo, places, each, amplitude);
        return 0;
    };
    using std::integral_constant;
    if (interleaved) {
        return wide ? launch(integral_constant<int, W>{}, std::false_type{}) : launch(integral_constant<int, 2>{}, std::false_type{});
    }
    return wide ? launch(integral_constant<int, W>{}, std::true_type{}) : launch(integral_constant<int, 1>{}, std::true_type{});
}

}  // namespace

// out[t, h * head_dim ..] = x[t, h * head_dim ..] turned by positions[t]; out may be x. Returns 0, a HIP error code, or -1 for sizes
// it refuses: head_dim even, 1 <= 2 * pairs <= head_dim, tokens * head_dim below 2^38 and 2^32 places in all.
extern "C" int mllm_rotary(const void* x, long long ldx, const int* positions, const unsigned long long* turns, int tokens, int pairs, int n_heads,
                           int head_dim, int interleaved, float amplitude, void* out, long long ldo, int dtype, hipStream_t stream) {
    if (tokens <= 0) return 0;
    if (n_heads < 1 || pairs < 1 || 2 * pairs > head_dim || head_dim % 2 != 0 || static_cast<long long>(tokens) * head_dim > 1ll << 38) return -1;
    const int rc = dtype == MLLM_F32 ? launch_rotary(static_cast<const float*>(x), ldx, positions, turns, tokens, pairs, n_heads, head_dim, interleaved, amplitude,
                                                     static_cast<float*>(out), ldo, stream)
                                     : launch_rotary(static_cast<const bf16_t*>(x), ldx, positions, turns, tokens, pairs, n_heads, head_dim, interleaved, amplitude,
                                                     static_cast<bf16_t*>(out), ldo, stream);
    if (rc != 0) return rc;
    MLLM_LAUNCH_CHECK();
    return 0;
}
