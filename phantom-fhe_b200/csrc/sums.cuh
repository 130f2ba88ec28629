// sums.cuh - products and sums of products of residues, as the position-by-position kernels form them, and vector access.
#pragma once
#include "modarith.cuh"
#include "ntt_kernels.cuh"

namespace b2 {

// ---- products of canonical residues ------------------------------------------------------------------------------------
// x y mod q by Barrett with one 64-bit quotient estimate: n = bit length of q, t = floor(x y / 2^(n-2)) < 2^(n+2),
// mu = floor(2^(62+n) / q) < 2^63; the estimate is short by one at most. Eight partial products instead of the sixteen of a
// 128-bit ratio.
__device__ __forceinline__ uint64_t mul_mod(uint64_t x, uint64_t y, const Mod &m) {
    const int n = 64 - __clzll((long long)m.q);
    const uint64_t lo = x * y, hi = __umul64hi(x, y);
    const uint64_t t = (hi << (66 - n)) | (lo >> (n - 2));
    return csub(lo - __umul64hi(t, m.mu) * m.q, m.q);
}

// the same for a sum of up to four products, q below 2^60: t < 2^64, the estimate is short by two at most
__device__ __forceinline__ uint64_t reduce_sum4(u128 x, const Mod &m) {
    const int n = 64 - __clzll((long long)m.q);
    const uint64_t t = (x.hi << (66 - n)) | (x.lo >> (n - 2));
    const uint64_t r = x.lo - __umul64hi(t, m.mu) * m.q;
    return csub(csub(r, 2 * m.q), m.q);
}

// ---- sums of products: how operands are held and summed, per prime class -------------------------------------------------
//   A, B     an operand as the sum wants it (split, or with its quotient); Acc the running sum; FLUSH how many terms it takes
//   flush    brings a full sum back to where it takes FLUSH terms again
//   finish   the canonical residue;  finish_mul the canonical residue times w
// Primes below 2^41: 21-bit pieces, four exact FP64 FMAs per term, no reduction until the end (a term adds less than 2^43).
struct SumFp21 {
    using F = ArithFp<false>;
    struct A {
        double l, h;
    };
    using B = A;
    struct K {
        F::K k;
        double w21, w42;  // 2^21, 2^42 mod q, least magnitude
    };
    struct Acc {
        double a0, a1, a2;
    };
    static constexpr int FLUSH = 120;
    __device__ __forceinline__ static K make(const Mod &m) {
        K r;
        r.k = F::make(m, 0);
        r.w21 = F::reduce(2097152.0, r.k), r.w42 = F::reduce(4398046511104.0, r.k);
        return r;
    }
    __device__ __forceinline__ static void zero(Acc &a) { a.a0 = a.a1 = a.a2 = 0.0; }
    __device__ __forceinline__ static A ld_a(uint64_t v, const K &) {
        return A{__dsub_rn(__longlong_as_double((long long)((v & 0x1FFFFF) | 0x4330000000000000ull)), FP_2_52),
                 __dsub_rn(__longlong_as_double((long long)((v >> 21) | 0x4330000000000000ull)), FP_2_52)};
    }
    __device__ __forceinline__ static B ld_b(uint64_t v, const K &k) { return ld_a(v, k); }
    __device__ __forceinline__ static void mac(Acc &s, const A &x, const B &y, const K &) {
        s.a0 = __fma_rn(x.l, y.l, s.a0);
        s.a1 = __fma_rn(x.l, y.h, __fma_rn(x.h, y.l, s.a1));
        s.a2 = __fma_rn(x.h, y.h, s.a2);
    }
    // a0 + a1 2^21 + a2 2^42, within 2 q + |a0|; |a1|, |a2| < 2^50
    __device__ __forceinline__ static double value(const Acc &s, const K &k) {
        const double u = F::mulmod(s.a1, F::Tw{k.w21, __dmul_rn(k.w21, k.k.qinv)}, k.k), v = F::mulmod(s.a2, F::Tw{k.w42, __dmul_rn(k.w42, k.k.qinv)}, k.k);
        return __dadd_rn(s.a0, __dadd_rn(u, v));
    }
    __device__ __forceinline__ static void flush(Acc &s, const K &k) { s = Acc{F::reduce(value(s, k), k.k), 0.0, 0.0}; }
    __device__ __forceinline__ static uint64_t finish(const Acc &s, const K &k) { return F::canon_fwd(value(s, k), k.k); }
    __device__ __forceinline__ static uint64_t finish_mul(const Acc &s, W2 w, const K &k) {
        const double wd = (double)w.w;
        return F::to_canon(F::mulmod(F::reduce(value(s, k), k.k), F::Tw{wd, __dmul_rn(wd, k.k.qinv)}, k.k), k.k);
    }
};
// Primes below 2^50: FP64 modular products (below 3/4 q in magnitude), summed up to 8 q = 2^53.
struct SumFp {
    using F = ArithFp<true>;
    using A = F::Tw;
    using B = double;
    using K = F::K;
    using Acc = double;
    static constexpr int FLUSH = 8;
    __device__ __forceinline__ static K make(const Mod &m) { return F::make(m, 0); }
    __device__ __forceinline__ static void zero(Acc &a) { a = 0.0; }
    __device__ __forceinline__ static A ld_a(uint64_t v, const K &k) {
        const double w = F::from_u64(v, k);
        return A{w, __dmul_rn(w, k.qinv)};
    }
    __device__ __forceinline__ static B ld_b(uint64_t v, const K &k) { return F::from_u64(v, k); }
    __device__ __forceinline__ static void mac(Acc &s, const A &x, B y, const K &k) { s = __dadd_rn(s, F::mulmod(y, x, k)); }
    __device__ __forceinline__ static void flush(Acc &s, const K &k) { s = F::reduce(s, k); }
    __device__ __forceinline__ static uint64_t finish(const Acc &s, const K &k) { return F::canon_fwd(s, k); }
    __device__ __forceinline__ static uint64_t finish_mul(const Acc &s, W2 w, const K &k) {
        return F::to_canon(F::mulmod(F::reduce(s, k), ld_a(w.w, k), k), k);
    }
};
// Primes below 2^60: 30-bit halves, four wide multiply-adds per term straight into 64-bit sums (two terms a sum of the
// middle weight, each below 2^60: sixteen fit), against four wide multiplies and eight carry instructions of a 128-bit sum.
struct SumInt30 {
    struct A {
        uint32_t l, h;
    };
    using B = A;
    using K = Mod;
    struct Acc {
        uint64_t s0, s1, s2;
        uint32_t s3;  // weights 2^0, 2^30, 2^60, 2^120
    };
    static constexpr int FLUSH = 8;
    __device__ __forceinline__ static K make(const Mod &m) { return m; }
    __device__ __forceinline__ static void zero(Acc &a) { a.s0 = a.s1 = a.s2 = 0, a.s3 = 0; }
    __device__ __forceinline__ static A ld_a(uint64_t v, const K &) { return A{(uint32_t)v & 0x3FFFFFFFu, (uint32_t)(v >> 30)}; }
    __device__ __forceinline__ static B ld_b(uint64_t v, const K &k) { return ld_a(v, k); }
    __device__ __forceinline__ static void mac(Acc &s, const A &x, const B &y, const K &) {
        s.s0 += (uint64_t)x.l * y.l;
        s.s1 += (uint64_t)x.l * y.h;
        s.s1 += (uint64_t)x.h * y.l;
        s.s2 += (uint64_t)x.h * y.h;
    }
    __device__ __forceinline__ static void carry(Acc &s) {
        s.s1 += s.s0 >> 30, s.s0 &= 0x3FFFFFFFu;
        s.s2 += s.s1 >> 30, s.s1 &= 0x3FFFFFFFu;
        s.s3 += (uint32_t)(s.s2 >> 60), s.s2 &= 0x0FFFFFFFFFFFFFFFull;
    }
    __device__ __forceinline__ static u128 total(Acc s) {
        carry(s);
        const uint64_t low = s.s0 | (s.s1 << 30);  // 60 bits
        return u128{low | (s.s2 << 60), (s.s2 >> 4) | ((uint64_t)s.s3 << 56)};
    }
    __device__ __forceinline__ static void flush(Acc &s, const K &k) {
        carry(s);
        if (s.s3 >= 128) {  // the sum nears 2^128
            const uint64_t r = barrett128(total(s), k.q, k.r0, k.r1);
            s = Acc{r & 0x3FFFFFFFu, r >> 30, 0, 0};
        }
    }
    __device__ __forceinline__ static uint64_t finish(const Acc &s, const K &k) { return barrett128(total(s), k.q, k.r0, k.r1); }
    __device__ __forceinline__ static uint64_t finish_mul(const Acc &s, W2 w, const K &k) { return mul_shoup(finish(s, k), w, k.q); }
};
// at most four terms: half the multiplications at the end
struct SumInt30Short : SumInt30 {
    __device__ __forceinline__ static uint64_t finish(const Acc &s, const K &k) { return reduce_sum4(total(s), k); }
    __device__ __forceinline__ static uint64_t finish_mul(const Acc &s, W2 w, const K &k) { return mul_shoup(finish(s, k), w, k.q); }
};
// Any prime up to 61 bits: 128-bit sums
struct SumInt {
    using A = uint64_t;
    using B = uint64_t;
    using K = Mod;
    using Acc = u128;
    static constexpr int FLUSH = 31;
    __device__ __forceinline__ static K make(const Mod &m) { return m; }
    __device__ __forceinline__ static void zero(Acc &a) { a = u128{0, 0}; }
    __device__ __forceinline__ static A ld_a(uint64_t v, const K &) { return v; }
    __device__ __forceinline__ static B ld_b(uint64_t v, const K &) { return v; }
    __device__ __forceinline__ static void mac(Acc &s, A x, B y, const K &) { mac128(s, x, y); }
    __device__ __forceinline__ static void flush(Acc &s, const K &k) { s = u128{barrett128(s, k.q, k.r0, k.r1), 0}; }
    __device__ __forceinline__ static uint64_t finish(const Acc &s, const K &k) { return barrett128(s, k.q, k.r0, k.r1); }
    __device__ __forceinline__ static uint64_t finish_mul(const Acc &s, W2 w, const K &k) { return mul_shoup(finish(s, k), w, k.q); }
};
template <class F>
__device__ __forceinline__ void with_sum(uint64_t q, F &&f) {
    if (q < FP_SMALL_LIMIT) f(SumFp21{});
    else if (q < FP_LIMIT) f(SumFp{});
    else if (q < INT_LAZY_LIMIT) f(SumInt30{});
    else f(SumInt{});
}

// ---- vector access: V = 4 words with 256-bit loads where every buffer is 32-byte aligned, two with 128-bit ones, else one word --
template <int V>
__device__ __forceinline__ void ldv(uint64_t (&x)[V], const uint64_t *p) {
    if constexpr (V == 4) {
        const u64x4 v = ld256(p);
        x[0] = v.a, x[1] = v.b, x[2] = v.c, x[3] = v.d;
    } else if constexpr (V == 2) {
        const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(p);
        x[0] = v.x, x[1] = v.y;
    } else {
        x[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void stv(uint64_t *p, const uint64_t (&x)[V]) {
    if constexpr (V == 4) st256(p, x[0], x[1], x[2], x[3]);
    else if constexpr (V == 2) *reinterpret_cast<ulonglong2 *>(p) = make_ulonglong2(x[0], x[1]);
    else *p = x[0];
}

}  // namespace b2
