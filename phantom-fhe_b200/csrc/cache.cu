// cache.cu - kernels and launchers of cache.cuh (a translation unit of its own: it compiles beside b200fhe.cu)
#include "cache.cuh"
#include "launch.cuh"
#include "sums.cuh"

namespace b2 {

// ---- pages ------------------------------------------------------------------------------------------------------------
// A thread owns the same 32 bytes of every page and walks its lane's steps, so that moves of a pool onto itself need no second
// buffer and no order between threads. Loads of a batch of steps go out before its stores: no step reads what an earlier step of
// the plan wrote, whichever is issued first. Steps of one source that follow one another read it once.
template <int CAP>
struct PageMoves {
    PageArgs a;
    uint16_t end[PAGE_LANES];
    PageStep step[CAP];
};

template <int COLS, int STEPS, int CAP>
__global__ void __launch_bounds__(256) pages_move_kernel(const __grid_constant__ PageMoves<CAP> m) {
    pdl_enter();
    const PageArgs &a = m.a;
    const uint32_t lane = blockIdx.y, c0 = (blockIdx.x * 256 * COLS + threadIdx.x) * 4;
    uint64_t *const pool = a.pool + (size_t)blockIdx.z * a.plane + c0;
    const uint64_t *src[COLS];
#pragma unroll
    for (int j = 0; j < COLS; j++)
        src[j] = a.src + (size_t)blockIdx.z * a.src_plane + c0 + j * 1024 + (c0 + j * 1024 >= a.half ? a.src_gap : 0);
    u64x4 kept[COLS];
    const uint32_t end = m.end[lane];
    for (uint32_t k = lane ? m.end[lane - 1] : 0; k < end; k += STEPS) {
        u64x4 v[STEPS][COLS];
        uint32_t from[STEPS];
#pragma unroll
        for (int u = 0; u < STEPS; u++) from[u] = k + u < end ? m.step[k + u].src : PAGE_KEPT;
#pragma unroll
        for (int u = 0; u < STEPS; u++) {
            const uint32_t s = from[u];
            if (u && s == from[u ? u - 1 : 0]) {
#pragma unroll
                for (int j = 0; j < COLS; j++) v[u][j] = v[u - 1][j];
            } else if (s < PAGE_KEPT) {
#pragma unroll
                for (int j = 0; j < COLS; j++) v[u][j] = ld256(src[j] + (size_t)s * a.src_page);
            } else {
#pragma unroll
                for (int j = 0; j < COLS; j++) v[u][j] = u64x4{0, 0, 0, 0};
            }
        }
#pragma unroll
        for (int u = 0; u < STEPS; u++) {
            if (k + u < end) {
                const uint32_t to = m.step[k + u].dst;
#pragma unroll
                for (int j = 0; j < COLS; j++) {
                    if (to == PAGE_KEPT) {
                        kept[j] = v[u][j];
                    } else {
                        const u64x4 x = from[u] == PAGE_KEPT ? kept[j] : v[u][j];
                        st256(pool + (size_t)to * a.page + j * 1024, x.a, x.b, x.c, x.d);
                    }
                }
            }
        }
    }
}

template <int CAP>
static void move_pages(const PageArgs &a, const PageStep *steps, const uint32_t *ends, uint32_t lanes, uint32_t planes, cudaStream_t s) {
    PageMoves<CAP> m;
    m.a = a;
    uint32_t longest = 0;
    for (uint32_t i = 0; i < lanes; i++) {
        m.end[i] = (uint16_t)ends[i];
        longest = std::max(longest, ends[i] - (i ? ends[i - 1] : 0));
    }
    std::copy_n(steps, ends[lanes - 1], m.step);
    const unsigned cols = a.half / 2;  // 32-byte columns of a page, a multiple of 2048
    const auto go = [&](auto kernel, unsigned per) { launch_k(kernel, dim3(cols / (256 * per), lanes, planes), 256, 0, s, m); };
    if (longest <= 1) go(pages_move_kernel<4, 1, CAP>, 4);
    else if (longest <= 4) go(pages_move_kernel<2, 4, CAP>, 2);
    else go(pages_move_kernel<1, 8, CAP>, 1);
}

void launch_pages_move(const PageArgs &a, const PageStep *steps, const uint32_t *ends, uint32_t lanes, uint32_t planes, cudaStream_t s) {
    if (ends[lanes - 1] <= PAGE_STEPS_FEW) move_pages<PAGE_STEPS_FEW>(a, steps, ends, lanes, planes, s);
    else move_pages<PAGE_STEPS>(a, steps, ends, lanes, planes, s);
}

// ---- sum of products of ciphertexts ------------------------------------------------------------------------------------
// out[g] = (sum_t a0 b0, sum_t a0 b1 + a1 b0, sum_t a1 b1) mod every prime: products of the pages with the scores that weigh them,
// summed before any of them is relinearised. A thread owns V positions of a limb and walks the terms; sums stay in registers as
// the prime's arithmetic likes them (sums.cuh) and are reduced once at the end. G queries share one read of the pages.
template <class S, int G, int V, int U>
__device__ __forceinline__ void multiply_sum_body(const SumArgs &a, const Mod &md) {
    const typename S::K k = S::make(md);
    const size_t N = (size_t)1 << a.logN;
    const uint32_t limb = blockIdx.y, i = (blockIdx.x * 128 + threadIdx.x) * V;
    const size_t o = (size_t)limb * N + i, ga = (size_t)a.la * N, gb = (size_t)a.lb * N;
    typename S::Acc acc[G][3][V];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int p = 0; p < 3; p++)
#pragma unroll
            for (int j = 0; j < V; j++) S::zero(acc[g][p][j]);
    int pending = 0;
    for (uint32_t t = 0; t < a.terms; t += U) {
        uint64_t b0[U][V], b1[U][V], a0[G][U][V], a1[G][U][V];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t + u < a.terms) {
                ldv<V>(b0[u], a.b[t + u] + o), ldv<V>(b1[u], a.b[t + u] + gb + o);
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const uint64_t *x = a.a[g * a.terms + t + u] + o;
                    ldv<V>(a0[g][u], x), ldv<V>(a1[g][u], x + ga);
                }
            }
        }
        // the middle sum takes two products a term
        if (pending + 2 * U > S::FLUSH) {
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int p = 0; p < 3; p++)
#pragma unroll
                    for (int j = 0; j < V; j++) S::flush(acc[g][p][j], k);
            pending = 0;
        }
        pending += 2 * U;
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (t + u < a.terms) {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    const typename S::A y0 = S::ld_a(b0[u][j], k), y1 = S::ld_a(b1[u][j], k);
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const typename S::B x0 = S::ld_b(a0[g][u][j], k), x1 = S::ld_b(a1[g][u][j], k);
                        S::mac(acc[g][0][j], y0, x0, k);
                        S::mac(acc[g][1][j], y1, x0, k);
                        S::mac(acc[g][1][j], y0, x1, k);
                        S::mac(acc[g][2][j], y1, x1, k);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int p = 0; p < 3; p++) {
            uint64_t *out = a.out + ((size_t)(g * 3 + p) * a.l) * N + o;
            uint64_t r[V];
#pragma unroll
            for (int j = 0; j < V; j++) r[j] = S::finish(acc[g][p][j], k);
            if (!a.first) {
                uint64_t was[V];
                ldv<V>(was, out);
#pragma unroll
                for (int j = 0; j < V; j++) r[j] = add_mod(r[j], was[j], md.q);
            }
            stv<V>(out, r);
        }
}

template <int G, int V, int U>
__global__ void __launch_bounds__(128) multiply_sum_kernel(const __grid_constant__ SumArgs a) {
    pdl_enter();
    const Mod md = a.mod[blockIdx.y];
    with_sum(md.q, [&](auto s) { multiply_sum_body<decltype(s), G, V, U>(a, md); });
}

void launch_multiply_sum(const SumArgs &a, uint32_t queries, cudaStream_t s) {
    const auto go = [&](auto kernel, unsigned v) { launch_k(kernel, dim3((1u << a.logN) / (128 * v), a.l), 128, 0, s, a); };
    switch (queries) {
        case 1: go(multiply_sum_kernel<1, 2, 2>, 2); break;
        case 2: go(multiply_sum_kernel<2, 1, 2>, 1); break;
        case 3: go(multiply_sum_kernel<3, 1, 2>, 1); break;
        default: go(multiply_sum_kernel<4, 1, 2>, 1); break;
    }
}

// ---- rotary positions ----------------------------------------------------------------------------------------------------
// theta[t][j] = position[t][axis[j]] inv_freq[j], rounded once, then (cos, sin) in every head of the position's block of slots.
// blockIdx.x = block of d_total slots (token), blockIdx.y = a share of its heads. A thread owns one slot of a head (in `rows` heads
// side by side where a head is shorter than the CTA), takes its sine and cosine once and stores them head after head.
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
