// Rotary positions: flash_rotary on rows of any tensor, and flash_append_paged, which turns new rows of K (and Q) on their way into the
// pages of a cache.
//
//   pair i of a row turns by angle = position * inv_freq[i]:  (a, b) -> factor * (a cos - b sin, a sin + b cos)
//
// The angle in turns, position * inv_freq / (2 pi), is worked out in 64 bits with the rounding errors of both products carried along, and cut to
// its fraction there: nothing is lost up to positions of 2^53.  Sine and cosine of what is left are taken in 32 bits.  (With products rounded
// to 32 bits the angle of position 10^6 is off by up to 0.03, to 64 bits that of 2^31 by 5e-7.)
//
// Bound by memory: every element is read once and written once.  A wave has one token: its lanes work out the token's sines
// and cosines, a pair each, into LDS of the wave's own, and then walk the rows (heads) of the token in pieces of a pair of 16-byte chunks, whose
// angles they read back from there.  So an angle costs its 64-bit products and its sine once per token, not once per head.  Tokens of
// short launches are shared out among `parts` waves.  Measured on one MI355X: rotary B4 H32 N4096 d128 bf16 43-52 us (5.2-6.2 TB/s read and
// written, a copy of that size 4.7-4.9), fp32 101 us (a copy 100), append of 16384 tokens H32 H_kv8 d128 with Q 79 us (5.1 TB/s), one token H32 2.2 us and 64 of them into
// their pages 4 us of GPU time (a launch).  (The rows' first pieces requested in front of the angles: d80 6.3 -> 6.1 us, but N4096 43.1 -> 47.4.)
#include "rotary_kernels.h"

namespace fa {
namespace {

typedef __bf16 bf16_t;

template <typename T, int N>
struct alignas(sizeof(T) * N) Piece {
    T e[N];
};

__device__ __forceinline__ int uniform_int(const int32_t* p)
{
    return *reinterpret_cast<const __attribute__((address_space(4))) int32_t*>(reinterpret_cast<uintptr_t>(p));
}
__device__ __forceinline__ int64_t uniform_position(const void* positions, int is64, int64_t at)
{
    if (is64) return *reinterpret_cast<const __attribute__((address_space(4))) int64_t*>(reinterpret_cast<uintptr_t>(static_cast<const int64_t*>(positions) + at));
    return uniform_int(static_cast<const int32_t*>(positions) + at);
}

constexpr int kMaxPairs = 256;  // FLASH limit on rot: 512
// 1 / (2 pi) as the sum of two
constexpr double kInvTwoPi = 0.15915494309189533577, kInvTwoPiLow = -9.839338337591243e-18;

// cosines and sines (times factor) of the token's pairs into cs[2 i], cs[2 i + 1]; `sign` -1 turns the other way
__device__ __forceinline__ void angles(const float* inv_freq, int pairs, int64_t position, float factor, float sign, int lane, FA_LDS float* cs)
{
    const double p = (double)position;
    for (int i = lane; i < pairs; i += 64) {
        const double w = (double)inv_freq[i], a = p * w, a_low = __builtin_fma(p, w, -a);
        const double whole = rint(a * kInvTwoPi);
        const float f = (float)(__builtin_fma(a, kInvTwoPi, -whole) + __builtin_fma(a, kInvTwoPiLow, a_low * kInvTwoPi));  // -0.5 ... 0.5
        float s, c;
        sincospif(2.0f * f, &s, &c);
        cs[2 * i] = c * factor;
        cs[2 * i + 1] = s * factor * sign;
    }
    // (LDS of the wave's own, and its operations complete in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T>
__device__ __forceinline__ void turn(T& a, T& b, float c, float s)
{
    const float x = (float)a, y = (float)b;
    a = (T)__builtin_fmaf(x, c, -(y * s));
    b = (T)__builtin_fmaf(x, s, y * c);
}

// Chunks of a row, W elements wide: first those that turn (`turning` of them: pairs of chunks rot / 2 apart, or, interleaved, chunks of W / 2
// pairs), then those that are copied.
template <int W, bool kInter>
__host__ __device__ __forceinline__ int turning_chunks(int rot)
{
    return kInter ? (W == 1 ? rot / 2 : rot / W) : rot / 2 / W;
}

template <typename T, int W, bool kInter>
__device__ __forceinline__ void do_chunk(const T* src, T* dst, int c, int turning, int rot, bool in_place, const FA_LDS float* cs)
{
    typedef Piece<T, W> P;
    if (c < turning) {
        if constexpr (kInter && W > 1) {
            P x = *reinterpret_cast<const P*>(src + c * W);
#pragma unroll
            for (int e = 0; e < W; e += 2) {
                const int i = (c * W + e) >> 1;
                turn(x.e[e], x.e[e + 1], cs[2 * i], cs[2 * i + 1]);
            }
            *reinterpret_cast<P*>(dst + c * W) = x;
        } else {
            const int ia = kInter ? 2 * c : c * W, ib = kInter ? 2 * c + 1 : c * W + rot / 2;
            P x = *reinterpret_cast<const P*>(src + ia), y = *reinterpret_cast<const P*>(src + ib);
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const int i = c * W + e;
                turn(x.e[e], y.e[e], cs[2 * i], cs[2 * i + 1]);
            }
            *reinterpret_cast<P*>(dst + ia) = x;
            *reinterpret_cast<P*>(dst + ib) = y;
        }
    } else if (!in_place) {
        const int at = rot + (c - turning) * W;
        *reinterpret_cast<P*>(dst + at) = *reinterpret_cast<const P*>(src + at);
    }
}

template <typename T, int W, bool kInter>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs a)
{
    __shared__ float table[4][2 * kMaxPairs];
    const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;
    const int64_t token = unit / a.parts;
    const int part = (int)(unit - token * a.parts);
    if (token >= (int64_t)a.B * a.N) return;
    const int b = a.by_n.quotient((int)token), n = (int)token - b * a.N;
    FA_LDS float* const cs = (FA_LDS float*)table[wave];
    angles(a.inv_freq, a.rot / 2, uniform_position(a.positions, a.positions_64, b * a.positions_batch + n), a.factor, a.inverse ? -1.0f : 1.0f, lane, cs);
    const T* const x = static_cast<const T*>(a.X) + b * a.x_batch + n * a.x_row;
    T* const y = static_cast<T*>(a.Y) + b * a.y_batch + n * a.y_row;
    const int turning = turning_chunks<W, kInter>(a.rot), chunks = turning + (a.d - a.rot) / W, items = a.H * chunks;
    const bool in_place = a.X == a.Y;
    for (int i = part * 64 + lane; i < items; i += a.parts * 64) {
        const int h = a.by_chunks.quotient(i), c = i - h * chunks;
        do_chunk<T, W, kInter>(x + h * a.x_head, y + h * a.y_head, c, turning, a.rot, in_place, cs);
    }
}

template <typename T, int W, bool kInter>
__global__ void __launch_bounds__(256) append_kernel(const AppendArgs a)
{
    __shared__ float table[4][128];  // d <= 128: up to 64 pairs
    const int lane = threadIdx.x & 63, wave = wave_uniform(threadIdx.x >> 6);
    const int unit = blockIdx.x * 4 + wave;
    const int token = unit / a.parts, part = unit - token * a.parts;
    if (token >= a.tokens) return;
    // sequence of the token: how many of the others begin at or in front of it
    int b = -1;
    for (int b0 = 0; b0 <= a.B; b0 += 64) {
        const int mine = b0 + lane;
        const uint64_t begun = __builtin_amdgcn_ballot_w64(mine <= a.B && a.cu[mine <= a.B ? mine : 0] <= token);
        b += __builtin_popcountll(begun);
        if (begun != ~0ull) break;
    }
    b = wave_uniform(b);
    if (b < 0 || b >= a.B) return;  // in front of the first sequence, behind the last
    const int c0 = uniform_int(a.cu + b), c1 = uniform_int(a.cu + b + 1);
    const int len = uniform_int(a.lens + b);
    const int64_t place = (int64_t)len - c1 + token;  // len - (c1 - c0) + (token - c0)
    (void)c0;
    FA_LDS float* const cs = (FA_LDS float*)table[wave];
    if (a.inv_freq)
        angles(a.inv_freq, a.rot / 2, a.positions ? uniform_position(a.positions, a.positions_64, token) : place, a.factor, 1.0f, lane, cs);
    const int turning = turning_chunks<W, kInter>(a.rot), chunks = turning + (a.d - a.rot) / W;
    auto rows = [&](const T* src, int64_t src_head, T* dst, int64_t dst_head, int heads, int first) __attribute__((always_inline)) {
        const int items = heads * chunks;
        const bool in_place = src == dst;
        for (int i = first * 64 + lane; i < items; i += a.parts * 64) {
            const int h = a.by_chunks.quotient(i), c = i - h * chunks;
            do_chunk<T, W, kInter>(src + h * src_head, dst + h * dst_head, c, turning, a.rot, in_place, cs);
        }
    };
    if (a.H > 0) rows(static_cast<const T*>(a.Q) + token * a.q_token, a.q_head, static_cast<T*>(a.O) + token * a.o_token, a.o_head, a.H, part);
    // a place that the sequence does not have, or a page that the cache does not have, is not written
    if (place < 0 || place >= a.capacity) return;
    const int in_table = a.by_page.quotient((int)place), row = (int)place - in_table * a.page;
    const int entry = uniform_int(a.table + (size_t)b * a.table_stride + in_table);
    if ((uint32_t)entry >= (uint32_t)a.num_pages) return;
    // (the waves of a token take turns: who has done more of Q's pieces begins further on)
    const int q_pieces = (a.H * chunks + 63) / 64, k_pieces = (a.Hk * chunks + 63) / 64;
    const int k_first = (part + a.parts - q_pieces % a.parts) % a.parts, v_first = (part + a.parts - (q_pieces + k_pieces) % a.parts) % a.parts;
    rows(static_cast<const T*>(a.K) + token * a.k_token, a.k_head, static_cast<T*>(a.K_cache) + entry * a.kc_page + row * a.kc_row, a.kc_head, a.Hk, k_first);
    const T* const v = static_cast<const T*>(a.V) + token * a.v_token;
    T* const vc = static_cast<T*>(a.V_cache) + entry * a.vc_page + row * a.vc_row;
    const int copy_chunks = a.d / 8;
    for (int i = v_first * 64 + lane; i < a.Hk * copy_chunks; i += a.parts * 64) {
        const int h = a.by_copy_chunks.quotient(i), c = i - h * copy_chunks;
        *reinterpret_cast<v4u*>(vc + h * a.vc_head + c * 8) = *reinterpret_cast<const v4u*>(v + h * a.v_head + c * 8);
    }
}

// Waves that keep the memory busy: 8 per CU.  (2048 / 4096 / 8192: append of 2620 tokens H16 H_kv4 d64 7.9 / 8.0 / 9.8 us, 512 tokens H32 H_kv8 d128
// 5.5 / 5.8 / 5.7, rotary B3 H12 N1777 d80 6.3 / 6.3 / 7.1.)
constexpr int kBusyWaves = 2048;

// waves per token: as many as there are pieces of 64 chunks, as long as the launch is short of waves
inline int parts_for(int64_t tokens, int64_t pieces)
{
    int64_t p = (kBusyWaves + tokens - 1) / tokens;
    if (p > pieces) p = pieces;
    return (int)(p < 1 ? 1 : p);
}

// elements that a thread moves at once: what the layout of the pairs allows of `wide`
inline int width_for(int wide, int d, int rot, bool inter)
{
    for (int w : {8, 4})
        if (w <= wide && (inter ? rot : rot / 2) % w == 0 && (d - rot) % w == 0) return w;
    return 1;
}

template <typename T, int W>
hipError_t launch_rotary_width(RotaryArgs a, hipStream_t st)
{
    const int turning = a.interleaved ? turning_chunks<W, true>(a.rot) : turning_chunks<W, false>(a.rot), chunks = turning + (a.d - a.rot) / W;
    const int64_t tokens = (int64_t)a.B * a.N;
    a.parts = parts_for(tokens, ((int64_t)a.H * chunks + 63) / 64);
    a.by_chunks = fast_div(chunks);
    const dim3 grid((unsigned)((tokens * a.parts + 3) / 4));
    return a.interleaved ? launch_kernel(rotary_kernel<T, W, true>, grid, dim3(256), 0, st, a)
                         : launch_kernel(rotary_kernel<T, W, false>, grid, dim3(256), 0, st, a);
}
template <typename T>
hipError_t launch_rotary_type(const RotaryArgs& a, int wide, hipStream_t st)
{
    const int w = width_for(wide, a.d, a.rot, a.interleaved != 0);
    return w == 8 ? launch_rotary_width<T, 8>(a, st) : w == 4 ? launch_rotary_width<T, 4>(a, st) : launch_rotary_width<T, 1>(a, st);
}

template <typename T, int W>
hipError_t launch_append_width(AppendArgs a, hipStream_t st)
{
    const int turning = a.interleaved ? turning_chunks<W, true>(a.rot) : turning_chunks<W, false>(a.rot), chunks = turning + (a.d - a.rot) / W;
    a.parts = parts_for(a.tokens, ((int64_t)a.H * chunks + 63) / 64 + ((int64_t)a.Hk * chunks + 63) / 64 + ((int64_t)a.Hk * (a.d / 8) + 63) / 64);
    a.by_chunks = fast_div(chunks);
    a.by_copy_chunks = fast_div(a.d / 8);
    const dim3 grid((unsigned)(((int64_t)a.tokens * a.parts + 3) / 4));
    return a.interleaved ? launch_kernel(append_kernel<T, W, true>, grid, dim3(256), 0, st, a)
                         : launch_kernel(append_kernel<T, W, false>, grid, dim3(256), 0, st, a);
}
template <typename T>
hipError_t launch_append_type(const AppendArgs& a, hipStream_t st)
{
    const int w = width_for(8, a.d, a.rot, a.interleaved != 0);
    return w == 8 ? launch_append_width<T, 8>(a, st) : w == 4 ? launch_append_width<T, 4>(a, st) : launch_append_width<T, 1>(a, st);
}

}  // namespace

int launch_rotary(const RotaryArgs& a, int dtype, int wide, hipStream_t st)
{
    RotaryArgs b = a;
    b.by_n = fast_div(a.N);
    return (int)(dtype == 0 ? launch_rotary_type<half_t>(b, wide, st) : dtype == 1 ? launch_rotary_type<bf16_t>(b, wide, st) : launch_rotary_type<float>(b, wide, st));
}

int launch_append(const AppendArgs& a, int dtype, hipStream_t st)
{
    AppendArgs b = a;
    b.by_page = fast_div(a.page);
    return (int)(dtype == 0 ? launch_append_type<half_t>(b, st) : launch_append_type<bf16_t>(b, st));
}

}  // namespace fa
