// nnrh_rotary.hip -- queries and keys turned by their tokens' positions: a pair
// (a, b) of a head's first `rotary` elements becomes
//   (a c - b s, b c + a s),   c, s = table[position][pair],
// in fp32, rounded once; the rest of a head is copied. Products and sums are
// rounded one by one (as the plain formula has them).
//
// Bound by memory: every element is read and written once. A thread has a vector
// of a head's elements and the one that it is paired with (or, neighbours being
// pairs, one vector), and their cosines and sines, which all heads of a token find
// in L1; nothing is shared between threads. 8191 tokens, 32 and 8 heads of 128, bf16:
// 172 MB in 33 us, 5.2 TB/s, a large copy's rate; 4 tokens 3.1 us, the launch.
#include "nnrh_decode.h"

#include <type_traits>

namespace nnrh {
namespace {

template <int TY> struct Elem { typedef float t; };
template <> struct Elem<FT_F16> { typedef _Float16 t; };
template <> struct Elem<FT_BF16> { typedef __bf16 t; };
template <class T, int V> struct Vec { typedef T t __attribute__((ext_vector_type(V))); };
template <class T> struct Vec<T, 1> { typedef T t; };

template <class T, int V>
__device__ __forceinline__ void load(const void* p, long long i, float* v) {
    const auto x = *(const typename Vec<T, V>::t*)((const T*)p + i);
    if constexpr (V == 1) {
        v[0] = (float)x;
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (float)x[j];
    }
}
template <class T, int V>
__device__ __forceinline__ void store(void* p, long long i, const float* v) {
    typename Vec<T, V>::t x;
    if constexpr (V == 1) {
        x = (T)v[0];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = (T)v[j];
    }
    *(typename Vec<T, V>::t*)((T*)p + i) = x;
}

// A unit is what a thread does: `turn` of a head's are of its turned elements, the
// rest of its `units` vectors that are copied.
struct RotaryUnits { uint32_t total, heads, turn, units; };

template <int TY, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(Rotary a, RotaryUnits n) {
    typedef typename Elem<TY>::t T;
    const uint32_t id = blockIdx.x * 256 + threadIdx.x;
    if (id >= n.total) return;
    const uint32_t row = id / n.units, u = id - row * n.units;
    const uint32_t tok = row / n.heads;
    int head = (int)(row - tok * n.heads);
    const uint32_t b = tok / (uint32_t)a.seq, t = tok - b * (uint32_t)a.seq;
    const int which = head >= a.r[0].heads;
    head -= which ? a.r[0].heads : 0;
    const RotaryRows r = which ? a.r[1] : a.r[0];
    const long long from = b * r.xb + t * r.xt + (long long)head * a.hd, to = b * r.yb + t * r.yt + (long long)head * a.hd;
    if (u >= n.turn) {
        const int e = a.rotary + (int)(u - n.turn) * V;
        *(typename Vec<T, V>::t*)((T*)r.y + to + e) = *(const typename Vec<T, V>::t*)((const T*)r.x + from + e);
        return;
    }
    const int pos = a.positions[tok];
    // neighbours as pairs come in one vector, or, one element a load, in two
    constexpr bool two = !INTER || V == 1;
    constexpr int NP = two ? V : V / 2;   // pairs
    const int half = a.rotary >> 1, p0 = (int)u * NP, e0 = INTER ? 2 * p0 : p0, step = INTER ? 1 : half;
    float x[2 * V], y[2 * V];
    load<T, V>(r.x, from + e0, x);
    if constexpr (two) load<T, V>(r.x, from + e0 + step, x + V);
    if (pos < 0) {   // padding: as it is
        store<T, V>(r.y, to + e0, x);
        if constexpr (two) store<T, V>(r.y, to + e0 + step, x + V);
        return;
    }
    const float2* cs = a.table + (long long)min(pos, a.held - 1) * half + p0;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        float2 w = cs[i];
        if (pos >= a.held) w = float2{__builtin_nanf(""), __builtin_nanf("")};
        const int lo = two ? i : 2 * i, hi = two ? V + i : 2 * i + 1;
        y[lo] = x[lo] * w.x - x[hi] * w.y;
        y[hi] = x[hi] * w.x + x[lo] * w.y;
    }
    store<T, V>(r.y, to + e0, y);
    if constexpr (two) store<T, V>(r.y, to + e0 + step, y + V);
}

template <int TY, int V, bool INTER>
hipError_t go(const Rotary& a, const RotaryUnits& n, hipStream_t s) {
    rotary_kernel<TY, V, INTER><<<(n.total + 255) / 256, 256, 0, s>>>(a, n);
    return hipGetLastError();
}
template <int TY, int V>
hipError_t by_pairs(const Rotary& a, bool in_place, hipStream_t s) {
    RotaryUnits n;
    n.heads = a.r[0].heads + a.r[1].heads;
    n.turn = a.interleaved && V > 1 ? a.rotary / V : a.rotary / 2 / V;
    n.units = n.turn + (in_place ? 0 : (a.hd - a.rotary) / V);
    n.total = (uint32_t)((long long)a.batch * a.seq * n.heads * n.units);
    if (!n.total) return hipSuccess;
    return a.interleaved ? go<TY, V, true>(a, n, s) : go<TY, V, false>(a, n, s);
}

}  // namespace

hipError_t launch_rotary(const Rotary& a, hipStream_t s) {
    if (a.batch == 0 || a.seq == 0) return hipSuccess;
    // the widest vectors, of 16 bytes at most, that divide every part of a row and its steps
    const long long part = a.interleaved ? a.rotary : a.rotary / 2;
    unsigned long long all = (unsigned long long)(part | (a.hd - a.rotary) | a.hd);
    uintptr_t at = 0;
    for (const RotaryRows& r : a.r) {
        all |= (unsigned long long)(r.xb | r.xt | r.yb | r.yt);
        at |= (uintptr_t)r.x | (uintptr_t)r.y;
    }
    const int es = float_type_size(a.type);
    all = all * es | at;
    // (the rest of a head is there already)
    const bool in_place = a.r[0].x == a.r[0].y && a.r[1].x == a.r[1].y;
    const auto of = [&](auto ty) {
        constexpr int TY = decltype(ty)::value, V = TY == FT_F32 ? 4 : 8;
        return all % 16 == 0 ? by_pairs<TY, V>(a, in_place, s)
             : all % 8 == 0 ? by_pairs<TY, V / 2>(a, in_place, s) : by_pairs<TY, 1>(a, in_place, s);
    };
    return a.type == FT_F32 ? of(std::integral_constant<int, FT_F32>{})
         : a.type == FT_F16 ? of(std::integral_constant<int, FT_F16>{}) : of(std::integral_constant<int, FT_BF16>{});
}

}  // namespace nnrh
