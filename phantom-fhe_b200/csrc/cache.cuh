// cache.cuh - operators of generation with an encrypted model: pages of a cache of ciphertexts, the value product over cached
// pages, rotary positions. Launchers of cache.cu; they set no error state of their own: the caller reads cudaGetLastError.
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "ntt_kernels.cuh"  // Mod
#include "page_plan.h"

namespace b2 {

// ---- pages: [plane][page][2][limbs][N] --------------------------------------------------------------------------------
constexpr int PAGE_STEPS = 480, PAGE_LANES = 64;
struct PageArgs {
    uint64_t *pool;
    const uint64_t *src;            // the pool itself, or another one at the same level or a higher one
    uint64_t page, src_page;        // words of a page
    uint64_t plane, src_plane;      // words of a plane
    uint32_t half;                  // words of a polynomial of the pool's level
    uint32_t src_gap;               // words by which a polynomial of the source is longer
};
// runs of steps for blockIdx.y = lane
void launch_pages_move(const PageArgs &a, const PageStep *steps, const uint32_t *lane_ends, uint32_t lanes, uint32_t planes, cudaStream_t s);

// ---- sum of products of ciphertexts -------------------------------------------------------------------------------------
constexpr int SUM_TERMS = 64, SUM_QUERIES = 4;
struct SumArgs {
    uint64_t *out;                  // [queries][3][l][N]
    const Mod *mod;
    uint32_t logN, l, la, lb;       // limbs: of the result, of a polynomial of the operands
    uint32_t terms, first;          // first: 0 adds to what out holds
    const uint64_t *b[SUM_TERMS];
    const uint64_t *a[SUM_QUERIES * SUM_TERMS];  // [query][terms]
};
void launch_multiply_sum(const SumArgs &a, uint32_t queries, cudaStream_t s);

// ---- sums of ciphertexts times plaintexts, several at once ----------------------------------------------------------------
constexpr int PLAIN_TERMS = 4, PLAIN_SETS = 32;
struct PlainSumArgs {
    uint64_t *out;                  // [sets][2][l][N]
    const Mod *mod;
    uint32_t logN, l, terms;
    const uint64_t *ct[PLAIN_SETS * PLAIN_TERMS];  // [set][terms], [2][l][N] each
    const uint64_t *pt[PLAIN_SETS * PLAIN_TERMS];  // [l][N]
};
void launch_multiply_plain_sum(const PlainSumArgs &a, uint32_t sets, cudaStream_t s);

// ---- rotary positions ---------------------------------------------------------------------------------------------------
enum { ROTARY_PAIRS = 0, ROTARY_HALVES = 1, ROTARY_INTERLEAVED = 2 };
struct RotaryArgs {
    double2 *out;                   // [1 or 3][ciphertexts][slots]
    const void *pos;                // [tokens][axes] with strides in elements
    const double *inv_freq;         // [pairs]
    const int32_t *axis;            // [pairs]
    const uint8_t *keep;            // [tokens], or null
    int64_t pos_t, pos_a, keep_t;
    double scaling;
    uint32_t tokens, heads, d_head, pairs, per, slots;  // per: positions of a ciphertext
    uint32_t cts, conjugate;
};
// pos_type: 0 int32, 1 int64, 2 float32, 3 float64
void launch_rotary_factors(const RotaryArgs &a, int packing, int pos_type, int sm_count, cudaStream_t s);

}  // namespace b2
