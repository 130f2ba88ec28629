// encoder.cuh - the CKKS encoder's device side (src/ckks.cu:68-190, src/fft.cu:90-346, src/rns_base.cu:49-240 in the
// reference): the "special" FFT over the rotation group generated by 5, the rounding of the scaled embedding to signed
// integer coefficients, and the CRT composition of a coefficient-form plaintext back to centred doubles.
//
// The transform is the one published with HEAAN (Cheon, Kim, Kim, Song): for n = N/2 slots, M = 2N, rot[j] = 5^j mod M and
// ksi[k] = exp(2 pi i k / M),
//   forward (coefficients -> slots): bit-reverse, then for len = 2, 4, .., n: butterflies (u, v) -> (u + w v, u - w v) on
//     the pairs (i + j, i + j + len/2), w = ksi[(rot[j] mod 4 len) * M / (4 len)];
//   inverse (slots -> coefficients): for len = n, .., 4, 2: (u, v) -> (u + v, (u - v) w) with
//     w = ksi[(4 len - rot[j] mod 4 len) * M / (4 len)], then bit-reverse and divide by n.
// Two launches over the whole vector, each running half of the stages on its sub-transforms in shared memory
// (cfft_pass_kernel); encoding rounds to coefficients in the second.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "modarith.cuh"
#include "ntt_kernels.cuh"  // Mod

namespace b2 {

__device__ __forceinline__ double2 cmul(double2 a, double2 b) {
    return make_double2(__fma_rn(a.x, b.x, -a.y * b.y), __fma_rn(a.x, b.y, a.y * b.x));
}

// The transform over the rotation group, n = 2^logn values, in two launches: a pass of 2^logT-point sub-transforms runs all
// its stages in shared memory (one launch per stage took 14 x 2 us at n = 2^14, with two dependent table loads in each). A CTA
// owns 1024 values: C = 1024 / T columns at distance n / T (STRIDED) or C contiguous runs of T. The twiddle of stage len at
// position j is ksi[r] of order 4 len, r = rot[j] mod 4 len (INVERSE: its conjugate); a thread does one butterfly per stage
// and has all its twiddles loaded before the first, so the two dependent loads are waited for once.
//   INVERSE (encode): strided pass (len = n .. 2 n / T), then the contiguous one, results bit-reversed and scaled;
//   forward (decode): contiguous pass on bit-reversed, scaled input, then the strided one.
// ROUND: the last inverse pass writes rint(Re) to coeffs[k] and rint(Im) to coeffs[k + n] instead of complex values.
// blockIdx.y: vector of a batch, one behind the other.
constexpr int CFFT_LOG_TILE = 10, CFFT_MAX_STAGES = 8;
template <bool INVERSE, bool STRIDED, bool ROUND>
__global__ void __launch_bounds__(512) cfft_pass_kernel(const double2 *in, double2 *out, int64_t *coeffs, uint32_t logn, uint32_t logT,
                                                        const uint32_t *__restrict__ rot, const double2 *__restrict__ ksi, double k) {
    pdl_enter();
    __shared__ double2 sm[1 << CFFT_LOG_TILE];
    in += (size_t)blockIdx.y << logn, out += (size_t)blockIdx.y << logn, coeffs += (size_t)blockIdx.y << (logn + 1);  // vector of a batch
    const uint32_t n = 1u << logn, log_other = logn - logT, logC = CFFT_LOG_TILE - logT, C = 1u << logC, T = 1u << logT;
    const uint32_t tid = threadIdx.x, tile = blockIdx.x;
    // shared position p of the tile <-> index of the transform: [e][c] strided, [c][e] contiguous
    auto index = [&](uint32_t p) { return STRIDED ? ((p >> logC) << log_other) + (tile << logC) + (p & (C - 1)) : (tile << CFFT_LOG_TILE) + p; };
    const uint32_t c = STRIDED ? tid & (C - 1) : tid >> (logT - 1), pr = STRIDED ? tid >> logC : tid & (T / 2 - 1);
    double2 w[CFFT_MAX_STAGES];
    {
        uint32_t r[CFFT_MAX_STAGES];
#pragma unroll
        for (int s = 0; s < CFFT_MAX_STAGES; s++) {
            if (s < (int)logT) {
                const uint32_t lh = INVERSE ? logT - 1 - s : s;  // log2 of the pair's distance in elements
                const uint32_t e = ((pr >> lh) << (lh + 1)) | (pr & ((1u << lh) - 1));
                const uint32_t idx = STRIDED ? (e << log_other) + (tile << logC) + c : e;
                r[s] = rot[idx & ((STRIDED ? 1u << (lh + log_other) : 1u << lh) - 1)];
            }
        }
#pragma unroll
        for (int s = 0; s < CFFT_MAX_STAGES; s++) {
            if (s < (int)logT) {
                const uint32_t lh = INVERSE ? logT - 1 - s : s, log_q = lh + (STRIDED ? log_other : 0) + 3;  // order 4 len = 8 times half of len
                const uint32_t q = r[s] & ((1u << log_q) - 1);
                w[s] = ksi[(size_t)(INVERSE ? (1u << log_q) - q : q) << (logn + 2 - log_q)];
            }
        }
    }
    for (uint32_t p = tid; p < (1u << CFFT_LOG_TILE); p += 512) {
        const uint32_t i = index(p);
        double2 x = in[!INVERSE && !STRIDED ? __brev(i) >> (32 - logn) : i];
        if (!INVERSE && !STRIDED) x = make_double2(x.x * k, x.y * k);
        sm[p] = x;
    }
#pragma unroll
    for (int s = 0; s < CFFT_MAX_STAGES; s++) {
        if (s < (int)logT) {
            const uint32_t lh = INVERSE ? logT - 1 - s : s;
            const uint32_t e = ((pr >> lh) << (lh + 1)) | (pr & ((1u << lh) - 1));
            const uint32_t p0 = STRIDED ? (e << logC) + c : (c << logT) + e, p1 = p0 + (STRIDED ? 1u << (lh + logC) : 1u << lh);
            __syncthreads();
            const double2 x = sm[p0], y = sm[p1];
            if (INVERSE) {
                sm[p0] = make_double2(x.x + y.x, x.y + y.y);
                sm[p1] = cmul(make_double2(x.x - y.x, x.y - y.y), w[s]);
            } else {
                const double2 t = cmul(y, w[s]);
                sm[p0] = make_double2(x.x + t.x, x.y + t.y);
                sm[p1] = make_double2(x.x - t.x, x.y - t.y);
            }
        }
    }
    __syncthreads();
    for (uint32_t p = tid; p < (1u << CFFT_LOG_TILE); p += 512) {
        const uint32_t i = index(p);
        double2 x = sm[p];
        if (INVERSE && !STRIDED) {
            const uint32_t o = __brev(i) >> (32 - logn);
            x = make_double2(x.x * k, x.y * k);
            if (ROUND) {
                coeffs[o] = __double2ll_rn(x.x);
                coeffs[o + n] = __double2ll_rn(x.y);
            } else {
                out[o] = x;
            }
        } else {
            out[i] = x;
        }
    }
}

// coefficient k = rint(Re u_k), coefficient k + n = rint(Im u_k); the caller has checked that |u| < 2^62
__global__ void __launch_bounds__(256) encode_round_kernel(const double2 *__restrict__ u, uint32_t n, int64_t *__restrict__ coeffs) {
    pdl_enter();
    const uint32_t k = blockIdx.x * blockDim.x + threadIdx.x;
    if (k >= n) return;
    const double2 x = u[k];
    coeffs[k] = __double2ll_rn(x.x);
    coeffs[k + n] = __double2ll_rn(x.y);
}

// CRT composition (src/rns_base.cu:173-234): residues res [l][N] in coefficient form -> the centred integer
// x in (-Q/2, Q/2], as a double times inv_scale; coefficient k goes to the real part of out[k], coefficient k + N/2 to the
// imaginary part. tab: hat [l][l] words (Q / q_i, little endian) | inv [l] ((Q/q_i)^-1 mod q_i) | Q [l] | half [l]
// (floor(Q / 2)). x = sum_i y_i (Q/q_i) - v Q with y_i = res_i inv_i mod q_i, everything in l + 1 words of 64 bits.
// v comes from a sum of y_i / q_i in FP64, at most one off (l <= 64 terms below 1, each within 2^-51), and is put right.
// The words live in registers: a kernel for every 8 words, each loop over the words unrolled. Bound by the latency of its carry
// chains (a thread per coefficient: a warp or two for a scheduler); with l a variable the words were in local memory and Q was
// subtracted up to l - 1 times: 9 limbs at N = 2^15 20.0 us, 16 at 2^16 65.5 us; 14.3 and 34.6 us so.
constexpr int B2_CRT_MAX_LIMBS = 64;
template <int L>
__global__ void __launch_bounds__(128) decode_compose_kernel(const uint64_t *__restrict__ res, const uint64_t *__restrict__ tab, const Mod *mod, uint32_t N,
                                                             uint32_t l, double inv_scale, double2 *__restrict__ out) {
    pdl_enter();
    extern __shared__ uint64_t crt_words[];
    for (uint32_t i = threadIdx.x; i < l * (l + 3); i += blockDim.x) crt_words[i] = tab[i];
    __syncthreads();
    const uint32_t n = blockIdx.x * blockDim.x + threadIdx.x;
    if (n >= N) return;
    const uint64_t *hat = crt_words, *inv = hat + l * l, *Q = inv + l, *half = Q + l;
    uint64_t acc[L], top_word = 0;  // words 0 .. l - 1, and word l
    double ratio = 0.0;             // x / Q
#pragma unroll
    for (int w = 0; w < L; w++) acc[w] = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < l; i++) {
        const Mod md = mod[i];
        u128 p{0, 0};
        mac128(p, res[(size_t)i * N + n], inv[i]);
        const uint64_t y = barrett128(p, md.q, md.r0, md.r1);
        ratio = __fma_rn((double)y, md.qinv, ratio);
        uint64_t carry = 0;
#pragma unroll
        for (int w = 0; w < L; w++) {
            if (w < (int)l) {
                // acc[w] + y * hat[i][w] + carry < 2^128
                const uint64_t h = hat[(size_t)i * l + w];
                uint64_t lo = y * h, hi = __umul64hi(y, h);
                lo += carry;
                hi += lo < carry;
                lo += acc[w];
                hi += lo < acc[w];
                acc[w] = lo;
                carry = hi;
            }
        }
        top_word += carry;
    }
    // acc - v Q, then back or on by one Q: word l says whether the difference is negative
    const uint64_t v = (uint64_t)ratio;
    uint64_t carry = 0, borrow = 0;
#pragma unroll
    for (int w = 0; w < L; w++) {
        if (w < (int)l) {
            uint64_t lo = v * Q[w], hi = __umul64hi(v, Q[w]);
            lo += carry;
            carry = hi + (lo < carry);
            const uint64_t x = acc[w];
            acc[w] = x - lo - borrow;
            borrow = x < lo || (x == lo && borrow);
        }
    }
    top_word -= carry + borrow;
    if ((int64_t)top_word < 0) {
        carry = 0;
#pragma unroll
        for (int w = 0; w < L; w++) {
            if (w < (int)l) {
                const uint64_t x = acc[w] + Q[w], y = x + carry;
                carry = (x < acc[w]) || (y < x);
                acc[w] = y;
            }
        }
        top_word += carry;
    }
    // whether acc >= Q, and (once it is below) acc > floor(Q / 2): by the sign of a difference
    bool ge = top_word != 0;
    if (!ge) {
        borrow = 0;
#pragma unroll
        for (int w = 0; w < L; w++)
            if (w < (int)l) borrow = acc[w] < Q[w] || (acc[w] == Q[w] && borrow);
        ge = !borrow;
    }
    if (ge) {
        borrow = 0;
#pragma unroll
        for (int w = 0; w < L; w++) {
            if (w < (int)l) {
                const uint64_t x = acc[w], q = Q[w];
                acc[w] = x - q - borrow;
                borrow = x < q || (x == q && borrow);
            }
        }
    }
    // centre: x > floor(Q/2) -> x - Q, kept as the magnitude Q - x and a sign
    borrow = 0;
#pragma unroll
    for (int w = 0; w < L; w++)
        if (w < (int)l) borrow = half[w] < acc[w] || (half[w] == acc[w] && borrow);
    const bool neg = borrow != 0;
    if (neg) {
        borrow = 0;
#pragma unroll
        for (int w = 0; w < L; w++) {
            if (w < (int)l) {
                const uint64_t x = Q[w], y = acc[w];
                acc[w] = x - y - borrow;
                borrow = x < y || (x == y && borrow);
            }
        }
    }
    // the two leading words carry more than the 53 bits a double keeps
    int top = 0;
    uint64_t lead = acc[0], next = 0;
#pragma unroll
    for (int w = 1; w < L; w++)
        if (w < (int)l && acc[w] != 0) top = w, lead = acc[w], next = acc[w - 1];
    double val = (double)lead;
    if (top > 0) val = __fma_rn(val, 18446744073709551616.0, (double)next);
    val = ldexp(val, 64 * (top > 0 ? top - 1 : 0)) * inv_scale;
    if (neg) val = -val;
    const uint32_t nh = N >> 1;
    double *o = reinterpret_cast<double *>(out + (n < nh ? n : n - nh));
    o[n < nh ? 0 : 1] = val;
}

template <class F>
static void with_crt_words(size_t l, F &&f) {
    if (l <= 8) f(decode_compose_kernel<8>);
    else if (l <= 16) f(decode_compose_kernel<16>);
    else if (l <= 24) f(decode_compose_kernel<24>);
    else if (l <= 32) f(decode_compose_kernel<32>);
    else if (l <= 48) f(decode_compose_kernel<48>);
    else f(decode_compose_kernel<64>);
}

}  // namespace b2
