// Attention within packed sequences where a sequence has few queries: tokens that are added to sequences.  16-bit, compiled once per head dim (-DEVO_D=32|64|96|128).
//
// Bound by memory: keys and values are read once and little is computed with them.  So the keys are split: a workgroup takes a chunk of one sequence's keys and one key head,
// its waves take 32 keys at a time each, and the queries of all heads that share the key head are the 16 columns of a matrix instruction (v_mfma_f32_16x16x32, S^T = K Q^T and O^T = V^T P^T as
// in packed_mfma.hip; more than 16 of them: 16 after 16).  A wave brings its keys and values into LDS of its own by the load path itself and waits for nobody: the next keys are asked for when
// the scores are formed, the next values when they have been multiplied; many waves with 16 KB (head dim 128) under way each are what memory's latency takes.  The waves' maxima, sums and
// outputs are joined in LDS; with more than one chunk to a sequence a second kernel joins the chunks', in their order.
//
// Which chunk: as for the tiles of packed_mfma.hip, chunk t of the launch belongs to the last segment j with key_begin(j) / chunk + j <= t, so that sequences of any lengths are spread evenly.
#include "packed_tiles.h"

namespace evo {

namespace EVO_CAT(packed_d, EVO_D) {

template <typename T> struct Mfma16;
template <> struct Mfma16<bf16_t> {
    static __device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Mfma16<f16_t> {
    static __device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

template <int NW, int CT> struct FewGeo {
    typedef PackedGeo::G G;
    static constexpr int KEYS = 32, ROWS = 16 * CT;                  // keys of a wave's step; columns
    static constexpr int ARRAY = KEYS * G::ROW, PIECES = ARRAY / 1024, RPP = 1024 / G::ROW;
    static constexpr int WAVES = NW;
    static constexpr int KS = EVO_D / 32, DT = EVO_D / 16;
    static constexpr int PITCH = EVO_D + 4;                          // of a joined row, fp32
    static constexpr int JOIN = WAVES * ROWS * (PITCH + 2) * 4;
    static constexpr int LDS = 2 * ARRAY * WAVES > JOIN ? 2 * ARRAY * WAVES : JOIN;
};
// Waves of a workgroup: 128 KB of LDS (head dim 32: 64), a CU's worth, where there are few workgroups; four where there are many, so that a CU has several and one does not wait for all of its waves.
constexpr int kFewWaves = PackedGeo::GD == 128 ? 8 : 16;

// CT: tiles of 16 columns that are multiplied with keys and values in LDS
template <typename T, bool PART, int NW, int CT>
__global__ void __launch_bounds__(NW * 64) packed_few(EvoPacked p, Parts parts) {
    typedef FewGeo<NW, CT> Few;
    typedef PackedGeo R;
    typedef R::G G;
    typedef typename Mfma<T>::v8 v8;
    typedef typename Mfma<T>::v4 v4;
    extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, gq = lane >> 4;
    const int group = p.H / p.Hk, D = p.D;
    const int hk = (int)(blockIdx.x % (unsigned)p.Hk), t = (int)(blockIdx.x / (unsigned)p.Hk);
    int j;
    const Segment s = find_segment<true>(p, [&](int begin, int x) { return begin / parts.chunk + x <= t; }, j);
    const int index = t - (s.k0 / parts.chunk + j);
    if (index < 0) return;
    const int64_t c0 = (int64_t)index * parts.chunk;
    const int nk = s.gap ? 0 : s.nk();
    if (c0 >= nk && (PART || index > 0)) return;
    // (none: zeros, by the only chunk; in scalar registers, where 64-bit comparisons are not formed by themselves)
    const int key_from = __builtin_amdgcn_readfirstlane((int)c0), key_to = __builtin_amdgcn_readfirstlane((int)min((int64_t)nk, c0 + parts.chunk));
    const int64_t rows = (int64_t)s.nq() * group;
    const int kst = (int)p.k_stride_t * 2, vst = (int)p.v_stride_t * 2;
    const char *kbase = (const char *)head_row<T>(p.k, s.k0, p.k_stride_t, hk, p.k_stride_h), *vbase = (const char *)head_row<T>(p.v, s.k0, p.v_stride_t, hk, p.v_stride_h);
    unsigned char *const kbuf = lds + wave * 2 * Few::ARRAY, *const vbuf = kbuf + Few::ARRAY;
    auto fetch = [&](const char *base, int stride, unsigned char *dst, int key) {
        const __amdgpu_buffer_rsrc_t rs = rows_at(base + (int64_t)key * stride, min(Few::KEYS, nk - key), stride, D);
#pragma unroll
        for (int i = 0; i < Few::PIECES; ++i) {
            const int r = i * Few::RPP + lane / G::C, c = (lane % G::C) ^ G::x(r);
            dma16(rs, dst + i * 1024, c * 8 < D ? r * stride + c * 16 : kFarOff);
        }
    };
    v8 one;
#pragma unroll
    for (int i = 0; i < 8; ++i) one[i] = (T)1.0f;
    const float c = p.scale * kLog2e;

    bool nan = false, none = false;   // (this thread has met): what is no number beside a sum of probabilities that is one; a sum of zero: every score lies below what the maximum begins with
    for (int64_t r0 = 0; r0 < rows; r0 += Few::ROWS) {
        // this lane's columns: a query and a head each
        int seen[CT];
        const T *q[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            const int64_t pr = min(r0 + 16 * ct + col, rows - 1);
            const int i = s.q0 + (int)(pr / group), h = hk * group + (int)(pr % group);
            seen[ct] = s.gap ? 0 : s.seen(i, p.causal);
            q[ct] = head_row<T>(p.q, i, p.q_stride_t, h, p.q_stride_h);
        }
        float m[CT], l[CT];
        f32x4 o[CT][Few::DT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            m[ct] = kMaskFloor;
            l[ct] = 0.0f;
#pragma unroll
            for (int dt = 0; dt < Few::DT; ++dt) o[ct][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        int key = key_from + wave * Few::KEYS;
        if (key < key_to) {
            fetch(kbase, kst, kbuf, key);
            fetch(vbase, vst, vbuf, key);
            v8 qf[CT][Few::KS];
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
                for (int ks = 0; ks < Few::KS; ++ks) qf[ct][ks] = ks * 32 + gq * 8 < D ? ld8(q[ct] + ks * 32 + gq * 8) : zero8<T>();
            }
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) asked_together<Few::KS>(qf[ct]);   // (waited for here, with the first keys and values: what is counted below are the rows' loads alone)
            for (;;) {
                const int next = key + Few::WAVES * Few::KEYS;
                const bool more = next < key_to;   // (uniform)
                wait_loads_but<Few::PIECES>();      // the keys (the values are younger)
                f32x4 a[CT][2];
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) a[ct][tt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int ks = 0; ks < Few::KS; ++ks) {
                        const v8 x = *reinterpret_cast<const v8 *>(kbuf + G::at(16 * tt + col, 4 * ks + gq));
#pragma unroll
                        for (int ct = 0; ct < CT; ++ct) a[ct][tt] = Mfma16<T>::mma(x, qf[ct][ks], a[ct][tt]);
                    }
                }
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the keys have been read
                if (more) fetch(kbase, kst, kbuf, next);
                v8 pf[CT];
#pragma unroll
                for (int ct = 0; ct < CT; ++ct) {
                    float top = -INFINITY;
#pragma unroll
                    for (int tt = 0; tt < 2; ++tt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            a[ct][tt][r] = key + 16 * tt + 4 * gq + r < seen[ct] ? a[ct][tt][r] : -INFINITY;
                            top = fmaxf(top, a[ct][tt][r]);
                        }
                    top = fmaxf(top, __shfl_xor(top, 16));
                    top = fmaxf(top, __shfl_xor(top, 32));
                    const float mn = fmaxf(m[ct], top * c), alpha = fast_exp2(m[ct] - mn);
                    m[ct] = mn;
#pragma unroll
                    for (int x = 0; x < 8; ++x) pf[ct][x] = (T)fast_exp2(fmaf(a[ct][x >> 2][x & 3], c, -mn));
                    l[ct] = dot8<T>(pf[ct], one, l[ct] * alpha);
#pragma unroll
                    for (int dt = 0; dt < Few::DT; ++dt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) o[ct][dt][r] *= alpha;
                }
                if (more) wait_loads_but<Few::PIECES>();   // the values (the next keys are younger)
                else wait_loads();
#pragma unroll
                for (int dt = 0; dt < Few::DT; ++dt) {
                    v8 vt;   // V^T: row 16 dt + col, the keys in the order in which a lane holds their probabilities
#pragma unroll
                    for (int h2 = 0; h2 < 2; ++h2) {
                        const int row = 16 * h2 + 4 * gq + (col >> 2), at = dt * 16 + 4 * (lane & 3);
                        const s16x4s w = __builtin_amdgcn_ds_read_tr16_b64_v4i16((s16x4s __attribute__((address_space(3))) *)(vbuf + G::at(row, at >> 3) + (at & 7) * 2));
                        const v4 x = __builtin_bit_cast(v4, w);
#pragma unroll
                        for (int y = 0; y < 4; ++y) vt[4 * h2 + y] = x[y];
                    }
#pragma unroll
                    for (int ct = 0; ct < CT; ++ct) o[ct][dt] = Mfma16<T>::mma(vt, pf[ct], o[ct][dt]);
                }
                if (!more) break;
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the values have been read
                fetch(vbase, vst, vbuf, next);
                key = next;
            }
        }
        // The waves' parts joined, every thread four columns of a row
        __syncthreads();
        float *const jo = reinterpret_cast<float *>(lds), *const jm = jo + Few::WAVES * Few::ROWS * Few::PITCH, *const jl = jm + Few::WAVES * Few::ROWS;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
            l[ct] += __shfl_xor(l[ct], 16);
            l[ct] += __shfl_xor(l[ct], 32);
            const int row = wave * Few::ROWS + 16 * ct + col;
#pragma unroll
            for (int dt = 0; dt < Few::DT; ++dt) *reinterpret_cast<f32x4 *>(jo + row * Few::PITCH + dt * 16 + gq * 4) = o[ct][dt];
            if (gq == 0) {
                jm[row] = m[ct];
                jl[row] = l[ct];
            }
        }
        __syncthreads();
        for (int jr = threadIdx.x / (EVO_D / 4), d = threadIdx.x % (EVO_D / 4) * 4; jr < Few::ROWS && r0 + jr < rows; jr += NW * 64 / (EVO_D / 4)) {
            float M = kMaskFloor, L = 0.0f;
#pragma unroll 4
            for (int w = 0; w < Few::WAVES; ++w) M = fmaxf(M, jm[w * Few::ROWS + jr]);
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int w = 0; w < Few::WAVES; ++w) {
                const float f = fast_exp2(jm[w * Few::ROWS + jr] - M);
                L = fmaf(jl[w * Few::ROWS + jr], f, L);
                const f32x4 x = *reinterpret_cast<const f32x4 *>(jo + (w * Few::ROWS + jr) * Few::PITCH + d);
#pragma unroll
                for (int y = 0; y < 4; ++y) sum[y] = fmaf(x[y], f, sum[y]);
            }
            const int64_t own = r0 + jr;
            const int oi = s.q0 + (int)(own / group), oh = hk * group + (int)(own % group);
            const int64_t row = (int64_t)oi * p.H + oh;
            if (PART) {
                const int64_t at = (int64_t)index * p.Tq * p.H + row;
                if (d < D) *reinterpret_cast<f32x4 *>(parts.o + at * D + d) = sum;
                if (d == 0) parts.ml[at] = make_float2(M, L);
            } else {
                const bool sees = nk > 0 && s.seen(oi, p.causal) > 0;
                const float inv = sees ? 1.0f / L : 0.0f;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    sum[y] = sees ? sum[y] * inv : 0.0f;
                    nan |= d < D && !(sum[y] == sum[y]) && L == L;
                }
                none |= sees && L == 0.0f;
                if (d < D) store4<T>((T *)p.o + row * D + d, sum[0], sum[1], sum[2], sum[3]);
                if (d < D && p.o_low) store4<T>((T *)p.o_low + row * D + d, left<T>(sum[0]), left<T>(sum[1]), left<T>(sum[2]), left<T>(sum[3]));
                if (d == 0 && p.lse) p.lse[(int64_t)oh * p.Tq + oi] = sees ? M + __log2f(L) : INFINITY;
            }
        }
        __syncthreads();
    }
    if constexpr (!PART) {
        if (!__syncthreads_or(nan || none)) return;
        // Some row holds something that is no number, perhaps because of keys that it does not see
        const bool below = __syncthreads_or(none);
        wait_loads();
        const EvoPacked late = parameters_again();
        for (int64_t x = wave; x < rows; x += Few::WAVES) {
            const int i = s.q0 + (int)(x / group), h = hk * group + (int)(x % group), seen = s.seen(i, late.causal);
            if (seen == 0 || all_finite<T>(late.o, (int64_t)late.H * late.D, h, late.D, i, i + 1, late.D)) continue;
            if (below || spoilt_forward<T>(late, s, hk, seen, nk)) row_forward<T>(late, s, i, h);
        }
    }
}

// The parts of a row joined: PER waves take every PER-th of them.
template <typename T, int PER>
__global__ void __launch_bounds__(PER > 4 ? PER * 64 : 256) packed_join(EvoPacked p, Parts parts, unsigned rows) {
    constexpr int WAVES = PER > 4 ? PER : 4, per = PER;
    __shared__ float sums[WAVES][128], rest[WAVES];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), own = wave % per;
    const unsigned row = blockIdx.x * (WAVES / per) + wave / per;
    const bool mine = row < rows;   // (uniform over the wave; over the workgroup where waves share a row)
    const int i = (int)(min(row, rows - 1) / (unsigned)p.H), h = (int)(min(row, rows - 1) % (unsigned)p.H), D = p.D;
    const Segment s = segment_of_row<false>(p, i);
    const int chunks = s.gap || s.seen(i, p.causal) == 0 ? 0 : parts.chunk ? min(parts.chunks, (s.nk() + parts.chunk - 1) / parts.chunk) : parts.chunks;
    const int64_t step = p.Tq * p.H;
    const float2 *ml = parts.ml + (int64_t)i * p.H + h;
    const float *o = parts.o + ((int64_t)i * p.H + h) * D;
    float M = kMaskFloor;
    for (int x = lane; x < chunks; x += 64) M = fmaxf(M, ml[x * step].x);
    M = wave_max(M);
    float L = 0.0f, a = 0.0f, b = 0.0f;
    const int d = min(lane * 2, D - 2);
#pragma unroll 8
    for (int x = own; x < chunks; x += per) {
        const float2 y = ml[x * step], z = *reinterpret_cast<const float2 *>(o + x * step * D + d);
        const float f = fast_exp2(y.x - M);
        L = fmaf(y.y, f, L);
        a = fmaf(z.x, f, a);
        b = fmaf(z.y, f, b);
    }
    if constexpr (per > 1) {
        sums[wave][lane * 2] = a;
        sums[wave][lane * 2 + 1] = b;
        if (lane == 0) rest[wave] = L;
        __syncthreads();
        if (own) return;
        for (int w = 1; w < per; ++w) {
            a += sums[w][lane * 2];
            b += sums[w][lane * 2 + 1];
            L += rest[w];
        }
    }
    if (!mine) return;
    const bool sees = !s.gap && s.seen(i, p.causal) > 0;
    const float inv = sees ? 1.0f / L : 0.0f;
    a = sees ? a * inv : 0.0f;
    b = sees ? b * inv : 0.0f;
    const bool used = lane * 2 < D;
    if (__any(used && (!(a == a) || !(b == b))) && L == L) {
        // (keys that are not seen: of a chunk all of them, else what other rows of a wave see, and the end of a stage)
        const EvoPacked late = parameters_again();
        const int seen = s.seen(i, late.causal), end = parts.chunk ? s.nk() : min(s.nk(), seen + 31 + 63);
        if (L == 0.0f || spoilt_forward<T>(late, s, h / (late.H / late.Hk), seen, end)) {
            row_forward<T, 4>(late, s, i, h);
            return;
        }
    }
    if (used) {
        T *out = (T *)p.o + ((int64_t)i * p.H + h) * D + lane * 2;
        typename Mfma<T>::v2 x;
        x[0] = (T)a;
        x[1] = (T)b;
        *reinterpret_cast<typename Mfma<T>::v2 *>(out) = x;
        if (p.o_low) {
            x[0] = (T)left<T>(a);
            x[1] = (T)left<T>(b);
            *reinterpret_cast<typename Mfma<T>::v2 *>((T *)p.o_low + ((int64_t)i * p.H + h) * D + lane * 2) = x;
        }
    }
    if (lane == 0 && p.lse) p.lse[(int64_t)h * p.Tq + i] = sees ? M + __log2f(L) : INFINITY;
}

template <typename T>
static int join(const EvoPacked &p, const Parts &parts, int64_t average, hipStream_t st) {
    const int64_t rows = p.Tq * p.H;
    if (average > 16) packed_join<T, 16><<<(unsigned)rows, 1024, 0, st>>>(p, parts, (unsigned)rows);
    else if (parts.chunks > 8) packed_join<T, 4><<<(unsigned)rows, 256, 0, st>>>(p, parts, (unsigned)rows);
    else packed_join<T, 1><<<(unsigned)((rows + 3) / 4), 256, 0, st>>>(p, parts, (unsigned)rows);
    return hip_rc();
}

// Keys of a chunk: as many as make some 256 workgroups of all sequences, keys and key heads (1024 of four waves), at least two (four) steps of every wave, since a workgroup that has only one spends its time
// on finding its place and joining; all of them where the longest sequence's walk, taken for up to four times the average's, is no longer than a second launch's way.  And not so few that the parts take
// more than kFewScratch bytes.
constexpr int64_t kFewScratch = 64 << 20;
struct FewPlan {
    Parts parts;
    bool many, wide;   // workgroups; columns
    size_t bytes;
};
static FewPlan few_plan(const EvoPacked &p, void *workspace) {
    FewPlan r;
    r.many = (int64_t)p.n * p.Hk >= 128;
    r.wide = p.Tq * (p.H / p.Hk) > (int64_t)16 * p.n;
    const int64_t unit = (r.many ? 4 : kFewWaves) * 32, room = (r.many ? 1024 : 256) / p.Hk - p.n, least = (r.many ? 4 : 2) * unit;
    const int64_t part = p.Tq * p.H * ((int64_t)p.D + 2) * (int64_t)sizeof(float), most = kFewScratch / (part ? part : 1);
    const int64_t longest = p.n < 4 ? p.Tk : 4 * p.Tk / p.n;
    int64_t chunk = room > 1 ? p.Tk / room : p.Tk;
    if (chunk < least) chunk = least;
    if (most > 1 && chunk < p.Tk / most + unit) chunk = p.Tk / most + unit;
    chunk = (chunk + unit / 2) / unit * unit;   // (to the nearest: workgroups that all CUs can begin at once)
    if (most < 2 || longest <= 5 * unit || chunk >= p.Tk) chunk = p.Tk < 1 ? unit : (p.Tk + unit - 1) / unit * unit;
    r.parts.chunk = (int)chunk;
    r.parts.chunks = (int)((p.Tk + chunk - 1) / chunk);
    r.parts.o = (float *)workspace;
    r.parts.ml = (float2 *)(r.parts.o + (int64_t)r.parts.chunks * p.Tq * p.H * p.D);
    r.bytes = r.parts.chunks > 1 ? (size_t)(r.parts.chunks * part) : 0;
    return r;
}

}  // namespace

size_t EVO_CAT(packed_few_bytes_d, EVO_D)(const EvoPacked &p) { return EVO_CAT(packed_d, EVO_D)::few_plan(p, nullptr).bytes; }
int EVO_CAT(launch_packed_few_d, EVO_D)(const EvoPacked &p, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    const FewPlan plan = few_plan(p, p.workspace);
    const Parts &parts = plan.parts;
    const int64_t grid = (p.Tk / parts.chunk + p.n + 2) * p.Hk, rows = p.Tq * p.H;
    if (parts.chunks > 1 && !grid_fits(rows, 1024)) return EVO_EOVERFLOW;   // (the join's)
    return by_half(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        auto go = [&](auto part, auto waves, auto tiles) {
            constexpr int NW = decltype(waves)::value, CT = decltype(tiles)::value, LDS = FewGeo<NW, CT>::LDS;
            constexpr auto kern = packed_few<T, decltype(part)::value, NW, CT>;
            static PerDevice done;
            if (!grid_fits(grid, NW * 64)) return (int)EVO_EOVERFLOW;
            if (const int rc = ensure_dynamic_lds((const void *)kern, LDS, done, nullptr)) return rc;
            kern<<<(unsigned)grid, NW * 64, LDS, st>>>(p, parts);
            const int rc = hip_rc();
            return rc || !decltype(part)::value ? rc : join<T>(p, parts, p.Tk / p.n / parts.chunk, st);
        };
        auto by_tiles = [&](auto part, auto waves) {
            return plan.wide ? go(part, waves, std::integral_constant<int, 2>()) : go(part, waves, std::integral_constant<int, 1>());
        };
        auto by_waves = [&](auto part) {
            return plan.many ? by_tiles(part, std::integral_constant<int, 4>()) : by_tiles(part, std::integral_constant<int, kFewWaves>());
        };
        return parts.chunks > 1 ? by_waves(std::true_type()) : by_waves(std::false_type());
    });
}
int EVO_CAT(launch_packed_join_d, EVO_D)(const EvoPacked &p, float *o, float2 *ml, int parts, hipStream_t st) {
    using namespace EVO_CAT(packed_d, EVO_D);
    return by_half(p.dtype, [&](auto t) { return join<decltype(t)>(p, Parts{o, ml, 0, parts}, parts, st); });
}

}  // namespace evo
