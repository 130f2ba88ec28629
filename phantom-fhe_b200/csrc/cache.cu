// cache.cu - kernels and launchers of cache.cuh (a translation unit of its own: it compiles beside b200fhe.cu)
#include "cache.cuh"
#include "launch.cuh"
#include "sums.cuh"

#include <type_traits>

namespace b2 {

// ---- pages ------------------------------------------------------------------------------------------------------------
// A thread owns the same 32 bytes of every page and walks its lane's steps, so that moves of a pool onto itself need no second
// buffer and no order between threads. Loads of a batch of steps go out before its stores: no step reads what an earlier step of
// the plan wrote, whichever is issued first. Steps of one source that follow one another in a batch read it once.
// Bound by HBM: a copy's rate, half reads and half writes. Four steps a batch take 56 registers, so that an SM has 1024 threads with
// 128 bytes each in flight: 47 pages of 2 MB in four planes change places in 121 us (6.5 TB/s); with eight steps (126 registers, 512
// threads) in 159, with two in 130.
struct PageMoves {  // 4 KB of parameters: they cost a launch less than 0.1 us over 256 bytes
    PageArgs a;
    uint16_t end[PAGE_LANES];
    PageStep step[PAGE_STEPS];
};

__global__ void __launch_bounds__(256, 4) pages_move_kernel(const __grid_constant__ PageMoves m) {
    pdl_enter();
    const PageArgs &a = m.a;
    const uint32_t lane = blockIdx.y, c0 = (blockIdx.x * 256 + threadIdx.x) * 4;
    uint64_t *const pool = a.pool + (size_t)blockIdx.z * a.plane + c0;
    const uint64_t *const src = a.src + (size_t)blockIdx.z * a.src_plane + c0 + (c0 >= a.half ? a.src_gap : 0);
    u64x4 kept = {0, 0, 0, 0};
    const uint32_t end = m.end[lane];
    for (uint32_t k = lane ? m.end[lane - 1] : 0; k < end; k += PAGE_BATCH) {
        u64x4 v[PAGE_BATCH];
        uint32_t from[PAGE_BATCH];
#pragma unroll
        for (int u = 0; u < PAGE_BATCH; u++) {
            const uint32_t s = from[u] = k + u < end ? m.step[k + u].src : PAGE_KEPT;
            if (u && s == from[u ? u - 1 : 0]) v[u] = v[u ? u - 1 : 0];
            else if (s < PAGE_KEPT) v[u] = ld256(src + (size_t)s * a.src_page);
            else v[u] = u64x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int u = 0; u < PAGE_BATCH; u++) {
            if (k + u < end) {
                const uint32_t to = m.step[k + u].dst;
                if (to == PAGE_KEPT) {
                    kept = v[u];
                } else {
                    const u64x4 x = from[u] == PAGE_KEPT ? kept : v[u];
                    st256(pool + (size_t)to * a.page, x.a, x.b, x.c, x.d);
                }
            }
        }
    }
}

void launch_pages_move(const PageArgs &a, const PageStep *steps, const uint32_t *ends, uint32_t lanes, uint32_t planes, cudaStream_t s) {
    PageMoves m;
    m.a = a;
    for (uint32_t i = 0; i < lanes; i++) m.end[i] = (uint16_t)ends[i];
    std::copy_n(steps, ends[lanes - 1], m.step);
    // 32-byte columns of a page: half / 2, a multiple of 2048
    launch_k(pages_move_kernel, dim3(a.half / 512, lanes, planes), 256, 0, s, m);
}

// ---- sum of products of ciphertexts ------------------------------------------------------------------------------------
// out[g] = (sum_t a0 b0, sum_t a0 b1 + a1 b0, sum_t a1 b1) mod every prime: products of the pages with the scores that weigh them,
// summed before any of them is relinearised. A thread owns one position of a limb and walks the terms, U of them loaded before the
// first is multiplied; sums stay in registers as the prime's arithmetic likes them (sums.cuh) and are reduced once at the end.
// G queries share one read of the pages, on primes of 2^50 and more two of them.
// Bound by HBM: 2 (G + 1) limbs a term for 3 G products. One word a thread and load keeps the sums of all arithmetics in 80 registers
// (G = 1; 768 threads an SM with sixteen loads each in flight): 32 terms at N = 2^16, 16 limbs of 40 bits take 161 to 165 us (1.10 GB, 6.7 to
// 6.8 TB/s), 17 terms of 6 limbs at 2^14 10 to 11 (some of it out of L2), with two words a thread 168 to 193. More queries take 128
// registers. How many terms they load at a time was chosen at one length, 24 pages of 12 limbs at 2^15, in one run: two queries (0.47 GB)
// 76.6 us with five terms (which spill 24 bytes), 77.4 with four, 80.5 with three; three (0.63 GB) 99.8 with four, 117 with three; four
// (0.79 GB) 126.8 with three, 129.3 with two; other runs have 78.5, 101.6 and 129.1. Four queries are where the power cap is felt: after
// two seconds of them 136.7 us (141.3 with four products a term in place of three). Sums of three and four queries are FP64 products: in
// 21-bit pieces, 72 registers of sums for four, 181 us; on integer primes, whose sums of 30-bit pieces are as wide, the queries go two by
// two over the same pages (55 bits: three 143 us, four 182 to 185; 187 to 259 at once). Two queries on 42 to 50 bits take 86.0 us, on 55
// bits 94.3. Terms dealt to four groups of threads that join
// in shared memory gain 1.3 us of 10 at 60 terms and 96 CTAs and lose everywhere else: not built.
constexpr int SUM_T = 128;

// FP64 products of primes below 2^41: 2048 of them stay below 2^53, so that no sum of a launch is brought back on the way
struct SumFpLong : SumFp {
    static constexpr int FLUSH = 2048;
};
static_assert(2 * SUM_TERMS <= SumFpLong::FLUSH);

// The middle sum takes (a0 + a1)(b0 + b1) and loses the two others at the end: three products a term instead of four.
//   both_a, both_b   the sum of two operands as an operand of S;  TERMS  how many terms the three sums take before they are brought back
// 21-bit pieces are added piece by piece (22 bits and 21: a term adds 2^44 to the two lower sums, sixty of them stay below 2^50); of
// FP64 residues below 2^50 one factor may be 2 q, the other is brought below q, and a product is below q; integers are reduced.
template <class S>
struct Pair {
    static constexpr int TERMS = S::FLUSH;
    __device__ __forceinline__ static typename S::A both_a(uint64_t x, uint64_t y, const typename S::A &, const typename S::A &, const Mod &md, const typename S::K &k) {
        return S::ld_a(add_mod(x, y, md.q), k);
    }
    __device__ __forceinline__ static typename S::B both_b(uint64_t x, uint64_t y, const typename S::B &, const typename S::B &, const Mod &md, const typename S::K &k) {
        return S::ld_b(add_mod(x, y, md.q), k);
    }
};
template <>
struct Pair<SumFp21> {
    using S = SumFp21;
    static constexpr int TERMS = 60;
    __device__ __forceinline__ static S::A both_a(uint64_t, uint64_t, const S::A &x, const S::A &y, const Mod &, const S::K &) {
        return S::A{__dadd_rn(x.l, y.l), __dadd_rn(x.h, y.h)};
    }
    __device__ __forceinline__ static S::B both_b(uint64_t, uint64_t, const S::B &x, const S::B &y, const Mod &, const S::K &) {
        return S::B{__dadd_rn(x.l, y.l), __dadd_rn(x.h, y.h)};
    }
};
template <class F>
struct PairFp {
    static constexpr int TERMS = F::FLUSH - 1;
    __device__ __forceinline__ static SumFp::A both_a(uint64_t x, uint64_t y, const SumFp::A &, const SumFp::A &, const Mod &md, const SumFp::K &k) {
        return SumFp::ld_a(add_mod(x, y, md.q), k);
    }
    __device__ __forceinline__ static SumFp::B both_b(uint64_t, uint64_t, const SumFp::B &x, const SumFp::B &y, const Mod &, const SumFp::K &) { return __dadd_rn(x, y); }
};
template <>
struct Pair<SumFp> : PairFp<SumFp> {};
template <>
struct Pair<SumFpLong> : PairFp<SumFpLong> {};

template <class S, int G, int U>
__device__ __forceinline__ void multiply_sum_body(const SumArgs &a, const Mod &md, uint32_t g0) {
    static_assert(U <= Pair<S>::TERMS);
    const typename S::K k = S::make(md);
    const size_t N = (size_t)1 << a.logN;
    const size_t o = (size_t)blockIdx.y * N + blockIdx.x * SUM_T + threadIdx.x, ga = (size_t)a.la * N, gb = (size_t)a.lb * N;
    typename S::Acc acc[G][3];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int p = 0; p < 3; p++) S::zero(acc[g][p]);
    int pending = 0;
    for (uint32_t t = 0; t < a.terms; t += U) {
        uint64_t b0[U], b1[U], a0[G][U], a1[G][U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t + u < a.terms) {
                b0[u] = a.b[t + u][o], b1[u] = a.b[t + u][gb + o];
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const uint64_t *x = a.a[(g0 + g) * a.terms + t + u] + o;
                    a0[g][u] = x[0], a1[g][u] = x[ga];
                }
            }
        }
        if (pending + U > Pair<S>::TERMS) {
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int p = 0; p < 3; p++) S::flush(acc[g][p], k);
            pending = 0;
        }
        pending += U;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t + u < a.terms) {
                const typename S::A y0 = S::ld_a(b0[u], k), y1 = S::ld_a(b1[u], k), y = Pair<S>::both_a(b0[u], b1[u], y0, y1, md, k);
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const typename S::B x0 = S::ld_b(a0[g][u], k), x1 = S::ld_b(a1[g][u], k);
                    S::mac(acc[g][0], y0, x0, k);
                    S::mac(acc[g][1], y, Pair<S>::both_b(a0[g][u], a1[g][u], x0, x1, md, k), k);
                    S::mac(acc[g][2], y1, x1, k);
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < G; g++) {
        uint64_t r[3];
#pragma unroll
        for (int p = 0; p < 3; p++) r[p] = S::finish(acc[g][p], k);
        r[1] = sub_mod(sub_mod(r[1], r[0], md.q), r[2], md.q);
#pragma unroll
        for (int p = 0; p < 3; p++) {
            uint64_t *out = a.out + (size_t)((g0 + g) * 3 + p) * a.l * N + o;
            *out = a.first ? r[p] : add_mod(r[p], *out, md.q);
        }
    }
}

template <int G, int U, int MIN_CTAS>
__global__ void __launch_bounds__(SUM_T, MIN_CTAS) multiply_sum_kernel(const __grid_constant__ SumArgs a) {
    pdl_enter();
    const Mod md = a.mod[blockIdx.y];
    if constexpr (G <= 2) {
        with_sum(md.q, [&](auto s) { multiply_sum_body<decltype(s), G, U>(a, md, 0); });
    } else if (md.q < FP_SMALL_LIMIT) {
        multiply_sum_body<SumFpLong, G, U>(a, md, 0);
    } else if (md.q < FP_LIMIT) {
        multiply_sum_body<SumFp, G, U>(a, md, 0);
    } else {
        with_sum(md.q, [&](auto s) {
            if constexpr (!std::is_same_v<decltype(s), SumFp> && !std::is_same_v<decltype(s), SumFp21>) {
                multiply_sum_body<decltype(s), 2, U>(a, md, 0);
                multiply_sum_body<decltype(s), G - 2, U>(a, md, 2);
            }
        });
    }
}

void launch_multiply_sum(const SumArgs &a, uint32_t queries, cudaStream_t s) {
    const dim3 grid((1u << a.logN) / SUM_T, a.l);
    switch (queries) {
        case 1: launch_k(multiply_sum_kernel<1, 4, 6>, grid, SUM_T, 0, s, a); break;
        case 2: launch_k(multiply_sum_kernel<2, 5, 4>, grid, SUM_T, 0, s, a); break;
        case 3: launch_k(multiply_sum_kernel<3, 4, 4>, grid, SUM_T, 0, s, a); break;
        default: launch_k(multiply_sum_kernel<4, 3, 4>, grid, SUM_T, 0, s, a); break;
    }
}

// ---- sums of ciphertexts times plaintexts ---------------------------------------------------------------------------------
// out[z] = sum_t ct[z][t] (.) pt[z][t], t below 4: what a rotated ciphertext is (x C + rot(x, s) A + rot(x, -s) B), for a batch of
// them in one launch. 3 limbs a term and 2 to read and write. Sixteen of three terms at 2^16, 16 limbs of 40 bits (1.48 GB) take 276 us,
// 5.3 TB/s; at 2^15, 12 limbs (0.55 GB) 107, on 55 bits 94 (5.9 TB/s, a copy has 6.46). Bound by what is in flight: 92 registers leave
// five CTAs an SM, each of which loads all its words, then multiplies, then stores.
template <class S>
__device__ __forceinline__ void plain_sum_body(const PlainSumArgs &a, const Mod &md) {
    const typename S::K k = S::make(md);
    const size_t N = (size_t)1 << a.logN, o = (size_t)blockIdx.y * N + (blockIdx.x * 128 + threadIdx.x) * 2, P = (size_t)a.l * N;
    const uint32_t z = blockIdx.z;
    typename S::Acc acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; i++) S::zero(acc[i][0]), S::zero(acc[i][1]);
    uint64_t x[PLAIN_TERMS][2], y[PLAIN_TERMS][2][2];
#pragma unroll
    for (int t = 0; t < PLAIN_TERMS; t++) {
        if (t < (int)a.terms) {
            ldv<2>(x[t], a.pt[z * a.terms + t] + o);
            const uint64_t *c = a.ct[z * a.terms + t] + o;
            ldv<2>(y[t][0], c), ldv<2>(y[t][1], c + P);
        }
    }
#pragma unroll
    for (int t = 0; t < PLAIN_TERMS; t++) {
        if (t < (int)a.terms) {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const typename S::A w = S::ld_a(x[t][j], k);
                S::mac(acc[0][j], w, S::ld_b(y[t][0][j], k), k);
                S::mac(acc[1][j], w, S::ld_b(y[t][1][j], k), k);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint64_t r[2] = {S::finish(acc[i][0], k), S::finish(acc[i][1], k)};
        stv<2>(a.out + (size_t)z * 2 * P + i * P + o, r);
    }
}
__global__ void __launch_bounds__(128) multiply_plain_sum_kernel(const __grid_constant__ PlainSumArgs a) {
    pdl_enter();
    const Mod md = a.mod[blockIdx.y];
    if (md.q < FP_LIMIT) plain_sum_body<SumFp>(a, md);
    else if (md.q < INT_LAZY_LIMIT) plain_sum_body<SumInt30Short>(a, md);
    else plain_sum_body<SumInt>(a, md);
}

void launch_multiply_plain_sum(const PlainSumArgs &a, uint32_t sets, cudaStream_t s) {
    launch_k(multiply_plain_sum_kernel, dim3((1u << a.logN) / 256, a.l, sets), 128, 0, s, a);
}

// ---- rotary positions ----------------------------------------------------------------------------------------------------
// theta[t][j] = position[t][axis[j]] inv_freq[j], rounded once, then (cos, sin) in every head of the position's block of slots.
// blockIdx.x = block of heads * d_head slots (token), blockIdx.y = a share of its heads. A thread owns one slot of a head (in `rows`
// heads side by side where a head is shorter than the CTA), takes its sine and cosine once and stores them head after head: a table in
// shared memory would save the `rows` - 1 others that take the same ones at the same time, and cost a barrier before the first store.
// Angles are doubles: position * inv_freq of a far position has no digits to spare in 32 bits. Bound by HBM, which takes the factors
// as they are written: 805 MB (4096 positions of 32 heads of 128, three vectors) in 116.6 us, 6.9 TB/s; 33.5 MB in 7.8 us, of which
// launch, positions and sines are 3.
template <class P, int PACKING>
__global__ void __launch_bounds__(256) rotary_factors_kernel(const __grid_constant__ RotaryArgs a) {
    pdl_enter();
    constexpr int VECS = PACKING == ROTARY_PAIRS ? 1 : 3;
    const uint32_t t = blockIdx.x, ct = t / a.per, block = t % a.per, width = a.heads * a.d_head;
    const size_t vec = (size_t)a.cts * a.slots;
    double2 *const out = a.out + (size_t)ct * a.slots + (size_t)block * width;
    const bool live = t < a.tokens && (!a.keep || a.keep[(int64_t)t * a.keep_t]);
    const uint32_t rows = a.d_head < 256 ? 256 / a.d_head : 1, row = a.d_head < 256 ? threadIdx.x / a.d_head : 0;
    const uint32_t h0 = (uint32_t)((uint64_t)a.heads * blockIdx.y / gridDim.y), h1 = (uint32_t)((uint64_t)a.heads * (blockIdx.y + 1) / gridDim.y);
    if (row < rows)
        for (uint32_t i = a.d_head < 256 ? threadIdx.x % a.d_head : threadIdx.x; i < a.d_head; i += 256) {
            double2 f[VECS];
#pragma unroll
            for (int v = 0; v < VECS; v++) f[v] = make_double2(0.0, 0.0);
            if (live) {
                const uint32_t j = PACKING == ROTARY_INTERLEAVED ? i / 2 : PACKING == ROTARY_HALVES && i >= a.pairs ? i - a.pairs : i;
                const bool second = PACKING == ROTARY_INTERLEAVED ? i & 1 : PACKING == ROTARY_HALVES && i >= a.pairs;
                if (j < a.pairs) {
                    const double theta = __dmul_rn((double)static_cast<const P *>(a.pos)[(int64_t)t * a.pos_t + a.axis[j] * a.pos_a], a.inv_freq[j]);
                    double sn, cs;
                    sincos(theta, &sn, &cs);
                    sn *= a.conjugate ? -a.scaling : a.scaling, cs *= a.scaling;
                    f[0] = make_double2(cs, VECS == 1 ? sn : 0.0);
                    if constexpr (VECS == 3) f[1].x = second ? 0.0 : -sn, f[2].x = second ? sn : 0.0;
                } else {
                    f[0].x = 1.0;
                }
            }
            for (uint32_t h = h0 + row; h < h1; h += rows)
#pragma unroll
                for (int v = 0; v < VECS; v++) out[v * vec + (size_t)h * a.d_head + i] = f[v];
        }
    // slots behind the last whole block
    if (block == a.per - 1 && blockIdx.y == 0)
        for (uint32_t i = a.per * width + threadIdx.x; i < a.slots; i += 256)
#pragma unroll
            for (int v = 0; v < VECS; v++) a.out[v * vec + (size_t)ct * a.slots + i] = make_double2(0.0, 0.0);
}

template <class P>
static void rotary(const RotaryArgs &a, int packing, dim3 grid, cudaStream_t s) {
    if (packing == ROTARY_PAIRS) launch_k(rotary_factors_kernel<P, ROTARY_PAIRS>, grid, 256, 0, s, a);
    else if (packing == ROTARY_HALVES) launch_k(rotary_factors_kernel<P, ROTARY_HALVES>, grid, 256, 0, s, a);
    else launch_k(rotary_factors_kernel<P, ROTARY_INTERLEAVED>, grid, 256, 0, s, a);
}

void launch_rotary_factors(const RotaryArgs &a, int packing, int pos_type, int sm_count, cudaStream_t s) {
    const unsigned blocks = a.cts * a.per, rows = a.d_head < 256 ? 256 / a.d_head : 1, most = (a.heads + rows - 1) / rows;
    // few positions: their heads are shared out until there are four CTAs an SM
    const unsigned parts = std::max(1u, std::min({most, 4u * (unsigned)sm_count / blocks, 65535u}));
    const dim3 grid(blocks, parts);
    switch (pos_type) {
        case 0: rotary<int32_t>(a, packing, grid, s); break;
        case 1: rotary<int64_t>(a, packing, grid, s); break;
        case 2: rotary<float>(a, packing, grid, s); break;
        default: rotary<double>(a, packing, grid, s); break;
    }
}

}  // namespace b2
