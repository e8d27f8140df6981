// Rotary positions: queries and keys turned pair by pair by angles that grow with their rows' positions, and the gradient, which is
// the turn back.
//
// The product of queries turned by a(i) and keys turned by a(j) depends on a(i) - a(j) alone.  An angle is position times frequency; in fp32 their product has lost
// all of its fraction of a turn from some 10^7 turns on and three digits of it at 10^4.  Here a frequency is the fraction of a turn per position as a
// 64-bit whole number, so that the product modulo 2^64 is the angle's fraction of a turn, exactly and for positions of either sign; its upper 32 bits are what sine and
// cosine are formed from (Taylor's polynomials over an eighth of a turn either way, 2e-9 off).
//
// Bound by memory: a row is read and written once.  A thread takes one vector of pairs (16 bytes where sizes, strides and addresses allow) of up to kHeads heads of
// a token, so that their sines are formed once and as many loads are under way.
#include "elements.h"
#include "kernels.h"

namespace evo {

constexpr int kRotaryHeads = 4;   // heads of a thread

struct RotaryGrid {
    unsigned total, units, pair_units, slices;   // threads; vectors of a row and those of them that are turned; threads that share a row's heads
};

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Vec { T v[VEC]; };

__device__ __forceinline__ void sincos_turn(uint64_t turn, float &s, float &c) {
    const unsigned u = (unsigned)(turn >> 32), quarter = (u + 0x20000000u) >> 30;
    const float a = (float)(int)(u - (quarter << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
    const float a2 = a * a;
    const float sn = a * fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 1.0f);
    const float cs = fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.0f);
    const float x = quarter & 1 ? cs : sn, y = quarter & 1 ? sn : cs;
    s = quarter & 2 ? -x : x;
    c = (quarter + 1) & 2 ? -y : y;
}

template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary(EvoRotary p, RotaryGrid g) {
    typedef Vec<T, VEC> V;
    constexpr int PAIRS = INTERLEAVED && VEC > 1 ? VEC / 2 : VEC;
    const unsigned id = blockIdx.x * 256u + threadIdx.x;
    if (id >= g.total) return;
    const unsigned u = id % g.units, row = id / g.units, slice = row % g.slices, t = row / g.slices;
    const unsigned n = t % (unsigned)p.N, bs = t / (unsigned)p.N, s = bs % (unsigned)p.S, b = bs / (unsigned)p.S;
    const bool turned = u < g.pair_units;
    float sn[PAIRS], cs[PAIRS];
    int64_t i, j;   // of this thread's first pair (copied values: i alone)
    if (turned) {
        const int64_t at = (int64_t)b * p.pos_stride_b + n;
        const int64_t pos = p.pos_bytes == 8 ? ((const int64_t *)p.pos)[at] : (int64_t)((const int *)p.pos)[at];
#pragma unroll
        for (int x = 0; x < PAIRS; ++x) {
            sincos_turn((uint64_t)pos * ((const uint64_t *)p.turns)[u * PAIRS + x], sn[x], cs[x]);
            sn[x] *= p.inverse ? -p.scale : p.scale;
            cs[x] *= p.scale;
        }
        i = INTERLEAVED ? (int64_t)u * PAIRS * 2 : (int64_t)u * VEC;
        j = INTERLEAVED ? i + 1 : i + p.R / 2;
    } else {
        i = j = (int64_t)p.R + (int64_t)(u - g.pair_units) * VEC;
    }
    const int heads = p.H + p.Hk;
    const T *src[kRotaryHeads];
    T *dst[kRotaryHeads];
    V a[kRotaryHeads], c[kRotaryHeads];
#pragma unroll
    for (int x = 0; x < kRotaryHeads; ++x) {
        const int h = (int)slice + x * (int)g.slices;
        if (h >= heads) break;
        const bool key = h >= p.H;
        const int64_t *in = key ? p.k_stride : p.q_stride, *out = key ? p.out_k_stride : p.out_q_stride;
        const int hh = key ? h - p.H : h;
        src[x] = (const T *)(key ? p.k : p.q) + b * in[0] + s * in[1] + n * in[2] + hh * in[3];
        dst[x] = (T *)(key ? p.out_k : p.out_q) + b * out[0] + s * out[1] + n * out[2] + hh * out[3];
        a[x] = *(const V *)(src[x] + i);
        if (!INTERLEAVED || VEC == 1) c[x] = *(const V *)(src[x] + j);
    }
#pragma unroll
    for (int x = 0; x < kRotaryHeads; ++x) {
        if ((int)slice + x * (int)g.slices >= heads) break;
        if (turned) {
            if (INTERLEAVED && VEC > 1) {
#pragma unroll
                for (int y = 0; y < PAIRS; ++y) {
                    const float v = (float)a[x].v[2 * y], w = (float)a[x].v[2 * y + 1];
                    a[x].v[2 * y] = (T)(v * cs[y] - w * sn[y]);
                    a[x].v[2 * y + 1] = (T)(w * cs[y] + v * sn[y]);
                }
            } else {
#pragma unroll
                for (int y = 0; y < VEC; ++y) {
                    const float v = (float)a[x].v[y], w = (float)c[x].v[y];
                    a[x].v[y] = (T)(v * cs[y] - w * sn[y]);
                    c[x].v[y] = (T)(w * cs[y] + v * sn[y]);
                }
                *(V *)(dst[x] + j) = c[x];
            }
        }
        *(V *)(dst[x] + i) = a[x];
    }
}

static bool rotary_fits(const EvoRotary &p, int vec, int es) {   // whether vectors of so many elements can be moved
    if (p.D % vec || (p.interleaved ? vec > 1 && p.R % vec : (p.R / 2) % vec)) return false;
    const int64_t *strides[] = {p.q_stride, p.out_q_stride, p.k_stride, p.out_k_stride};
    const void *ptrs[] = {p.q, p.out_q, p.k, p.out_k};
    for (int i = 0; i < (p.Hk ? 4 : 2); ++i) {
        if ((uintptr_t)ptrs[i] % (vec * es)) return false;
        for (int d = 0; d < 4; ++d)
            if (strides[i][d] % vec) return false;
    }
    return true;
}

template <typename T>
static int launch_rotary(const EvoRotary &p, hipStream_t st) {
    constexpr int es = sizeof(T);
    int vec = 16 / es;
    while (vec > 1 && !rotary_fits(p, vec, es)) vec /= 2;
    const int64_t tokens = (int64_t)p.B * p.S * p.N, heads = (int64_t)p.H + p.Hk;
    RotaryGrid g;
    g.pair_units = p.interleaved && vec > 1 ? p.R / vec : p.R / 2 / vec;
    g.units = g.pair_units + (p.D - p.R) / vec;
    if ((double)tokens * (double)heads * (double)g.units > 1e18) return EVO_EOVERFLOW;
    // A head to a thread where there are too few of them to fill the chip otherwise
    const int64_t rows = tokens * heads, threads = rows * g.units;
    g.slices = (unsigned)(threads > 256 * 1024 ? (heads + kRotaryHeads - 1) / kRotaryHeads : heads);
    const int64_t total = tokens * g.slices * g.units;
    if (!grid_fits((total + 255) / 256, 256)) return EVO_EOVERFLOW;
    g.total = (unsigned)total;
    const unsigned grid = (unsigned)((total + 255) / 256);
    auto go = [&](auto v, auto il) {
        rotary<T, decltype(v)::value, decltype(il)::value><<<grid, 256, 0, st>>>(p, g);
        return hip_rc();
    };
    auto by_layout = [&](auto v) { return p.interleaved ? go(v, std::true_type()) : go(v, std::false_type()); };
    switch (vec) {
        case 8: if constexpr (es == 2) return by_layout(std::integral_constant<int, 8>());
        case 4: return by_layout(std::integral_constant<int, 4>());
        case 2: return by_layout(std::integral_constant<int, 2>());
        default: return by_layout(std::integral_constant<int, 1>());
    }
}

}  // namespace evo

extern "C" int evoattn_rotary(const EvoRotary *p, void *hip_stream) {
    using namespace evo;
    if (!p || p->B < 0 || p->S < 0 || p->N < 0 || p->H < 0 || p->Hk < 0 || p->D < 1 || p->R < 2 || p->R % 2 || p->R > p->D || !known_dtype(p->dtype) ||
        (p->pos_bytes != 4 && p->pos_bytes != 8))
        return EVO_EINVAL;
    if (!p->B || !p->S || !p->N || (!p->H && !p->Hk)) return EVO_OK;
    if (!p->pos || !p->turns || (p->H && (!p->q || !p->out_q)) || (p->Hk && (!p->k || !p->out_k))) return EVO_EINVAL;
    if ((int64_t)p->B * p->S > UINT32_MAX || (int64_t)p->B * p->S * p->N > UINT32_MAX || (int64_t)p->H + p->Hk > INT32_MAX / 64 || p->D > 65536) return EVO_EOVERFLOW;
    return by_dtype(p->dtype, [&](auto t) { return launch_rotary<decltype(t)>(*p, (hipStream_t)hip_stream); });
}
