// encoder.hip.h -- what the sequence-encoder kernels share: element types on the matrix
// cores, swizzled tiles in LDS, the dropout generator, the relative position bias.
//
// Products run on the 32x32 MFMA forms.  A fragment is 16 bytes a lane, a "chunk" of one
// row of a tile: lane l holds row l % 32 and chunk 2 s + l / 32 of step s (8 elements of
// 16 bits for one 32x32x16 MFMA; 4 of 32 bits for four 32x32x2 MFMAs, element e of both
// half waves in the e-th).  Accumulator v of lane l is row 8 (v / 4) + 4 (l / 32) + v % 4,
// column l % 32.
//
// A product's result can be the next one's operand without leaving its lanes: a sum over
// the rows may run in any order, so step f of it takes the rows that a lane holds in
// consecutive accumulators, and the other operand is read from LDS in the same order
// (frag_t below).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "capi_util.hip.h"
#include "../../include/d2p_amd_encoder.h"

namespace d2p_amd {
namespace enc {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef float f4v __attribute__((ext_vector_type(4)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));
typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8v __attribute__((ext_vector_type(8)));
typedef __bf16 b8v __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.4426950408889634f;
constexpr unsigned OOB = 0x80000000u;   // an offset past every resource's records

template <class T, class U> __device__ __forceinline__ T bits(U x) {
    return __builtin_bit_cast(T, x);
}

// ---------------------------------------------------------------------------
// element types
// ---------------------------------------------------------------------------
template <class T> struct Elem;

template <> struct Elem<float> {
    static constexpr int PER = 4;   // elements of a chunk
    static __device__ __forceinline__ f16v mma(u4v a, u4v b, f16v c) {
        const f4v x = bits<f4v>(a), y = bits<f4v>(b);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
    // accumulators PER f .. of a result, as the fragment of step f of the next product
    static __device__ __forceinline__ u4v pack(const float* p) {
        return bits<u4v>(f4v{p[0], p[1], p[2], p[3]});
    }
    static __device__ __forceinline__ void unpack(u4v c, float* x) {
        const f4v v = bits<f4v>(c);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    }
    static __device__ __forceinline__ float load(const void* p, long long i) {
        return ((const float*)p)[i];
    }
    static __device__ __forceinline__ void store(void* p, long long i, float v) {
        ((float*)p)[i] = v;
    }
    // four neighbours, 16 bytes
    static __device__ __forceinline__ void store4(void* p, const float* v) {
        *(f4v*)p = f4v{v[0], v[1], v[2], v[3]};
    }
};

template <class E, class V8, class V4> struct Elem16 {
    static constexpr int PER = 8;
    static __device__ __forceinline__ u4v pack(const float* p) {
        V8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (E)p[e];
        return bits<u4v>(v);
    }
    static __device__ __forceinline__ void unpack(u4v c, float* x) {
        const V8 v = bits<V8>(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
    }
    static __device__ __forceinline__ float load(const void* p, long long i) {
        return (float)((const E*)p)[i];
    }
    static __device__ __forceinline__ void store(void* p, long long i, float v) {
        ((E*)p)[i] = (E)v;
    }
    // four neighbours, 8 bytes
    static __device__ __forceinline__ void store4(void* p, const float* v) {
        V4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (E)v[e];
        *(u2v*)p = bits<u2v>(x);
    }
};

typedef _Float16 h4v __attribute__((ext_vector_type(4)));
typedef __bf16 b4v __attribute__((ext_vector_type(4)));

template <> struct Elem<_Float16> : Elem16<_Float16, h8v, h4v> {
    static __device__ __forceinline__ f16v mma(u4v a, u4v b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(bits<h8v>(a), bits<h8v>(b), c, 0, 0, 0);
    }
};
template <> struct Elem<__bf16> : Elem16<__bf16, b8v, b4v> {
    static __device__ __forceinline__ f16v mma(u4v a, u4v b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(bits<b8v>(a), bits<b8v>(b), c, 0, 0, 0);
    }
};

// ---------------------------------------------------------------------------
// tiles
// ---------------------------------------------------------------------------
// A tile of rows of DP features lies in LDS row by row, chunk c of row r at slot
// c ^ swz(r) of the row.  Sixteen rows' equal chunks (an operand's rows) and four rows'
// four neighbouring chunks (a transposed operand's) then each cover the 64 banks once.
// (96 features lie in rows of 128.)
template <class T, int DP> struct Tile {
    static constexpr int PER = Elem<T>::PER;
    static constexpr int NCH = (DP == 96 ? 128 : DP) / PER;   // chunks of a row
    static constexpr int ROW = NCH * 16;          // bytes of a row
    static constexpr int STEPS = DP / PER / 2;    // MFMA steps over the features
    static constexpr int FRAGS = 32 / (2 * PER);  // MFMA steps over 32 rows
    static constexpr int bytes(int rows) { return rows * NCH * 16; }

    static __device__ __forceinline__ int swz(int r) {
        if (NCH >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        if (NCH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        return (r >> 2) & 3;
    }
    static __device__ __forceinline__ int slot(int row, int c) {
        return row * NCH + (c ^ swz(row));
    }
    // Fragments.  A lane's place in a tile is one number of bytes, row_at or col_at; the rest of
    // an address is constants: chunks and the swizzle's share of a row number are combined
    // with it by exclusive or (they touch only the bits of the chunk), the row by an offset.
    static __device__ __forceinline__ int row_at(int lane) {
        return 16 * slot(lane & 31, lane >> 5);
    }
    // rows row0 .. row0 + 31 (row0 a multiple of 32) as an operand's rows, step s over the
    // features
    static __device__ __forceinline__ u4v frag(const u4v* tile, int row0, int s, int ra) {
        return *(const u4v*)((const char*)tile + row0 * ROW + (ra ^ (32 * s)));
    }
    static __device__ __forceinline__ int col_at(int lane) {
        const int h = lane >> 5;
        if (PER == 4)
            return 16 * slot(4 * h, (lane & 31) >> 2) + 4 * (lane & 3);
        return 16 * slot(4 * h + ((lane >> 2) & 3), 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) +
               8 * (lane & 1);
    }
    // features d0 .. d0 + 31 as an operand's rows, step f over rows row0 .. row0 + 31 in
    // the order of the accumulators: half wave h takes rows 8 g + 4 h + 0 .. 3 of
    // f = g (32 bits) or g = 2 f, 2 f + 1 (16 bits: ds_read_b64_tr_b16 gives each of 16
    // lanes one column of four rows)
    static __device__ __forceinline__ u4v frag_t(const u4v* tile, int row0, int d0, int f,
                                                 int ca) {
        const char* t = (const char*)tile + row0 * ROW;
        if constexpr (PER == 4) {
            u4v x;
#pragma unroll
            for (int r = 0; r < 4; ++r)
                x[r] = *(const unsigned*)(t + (8 * f + r) * ROW +
                                          (ca ^ (4 * d0) ^ (16 * swz(8 * f + r))));
            return x;
        } else {
            s4v x[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const char* q = t + (16 * f + 8 * n) * ROW + (ca ^ (2 * d0) ^ (16 * swz(8 * n)));
                x[n] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s4v*)q);
            }
            const u2v a = bits<u2v>(x[0]), b = bits<u2v>(x[1]);
            return u4v{a.x, a.y, b.x, b.y};
        }
    }
};

// raw buffer over `bytes` bytes from base: loads past its end give 0
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* base, long long n) {
    const int m = (int)(n < 0 ? 0 : n > 0x7fffffffLL ? 0x7fffffffLL : n);
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, m, 0x00020000);
}

// The rows of one head: row r of `rows` at base + r * stride bytes, `chunks` chunks each.
struct Rows {
    const char* base;
    long long stride;
    int rows, chunks;
    // from row r0 on; a row past the last is out of range (stride >= a row's bytes)
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t from(int r0) const {
        const long long left = rows - r0;
        return rsrc(base + r0 * stride, left > 0 ? (left - 1) * stride + chunks * 16 : 0);
    }
    __device__ __forceinline__ unsigned at(int r, int c) const {
        return c < chunks ? (unsigned)r * (unsigned)stride + (unsigned)c * 16u : OOB;
    }
};

// One tile of R rows straight from memory to LDS, by the waves of a workgroup together: an
// instruction brings 64 chunks to consecutive slots, and each lane fetches the chunk that
// belongs in its slot.  Out of range (past the last row, past D) comes as zeros.  Inline
// assembly, so that the compiler does not make every later LDS read wait for it: wait_dma()
// and a barrier do, one tile later.  M0 takes the LDS address; the compiler uses M0 for
// nothing here.  (Five wait states lie between a vector instruction that writes a scalar
// register and a load that takes its resource from there; the compiler does not look into
// the assembly to place them.)
template <class T, int DP, int R, int NW> struct TileDma {
    using TL = Tile<T, DP>;
    static constexpr int INSTR = R * TL::NCH / 64, COUNT = (INSTR + NW - 1) / NW;
    static constexpr int ROWS = 64 / TL::NCH;   // of an instruction
    unsigned off[COUNT];
    __device__ __forceinline__ void init(const Rows& src, int wave, int lane) {
#pragma unroll
        for (int n = 0; n < COUNT; ++n) {
            const int r = (wave + NW * n) * ROWS + lane / TL::NCH;
            off[n] = src.at(r, (lane % TL::NCH) ^ TL::swz(r));
        }
    }
    __device__ __forceinline__ void issue(const Rows& src, int r0, const u4v* tile,
                                          int wave) const {
        const long long left = ((long long)src.rows - r0 - 1) * src.stride + src.chunks * 16;
        const unsigned n = src.rows <= r0 ? 0u : left > 0x7fffffffLL ? 0x7fffffffu : (unsigned)left;
        const uint64_t b = (uint64_t)(src.base + (long long)r0 * src.stride);
        const u4v r = {(unsigned)__builtin_amdgcn_readfirstlane((unsigned)b),
                       (unsigned)__builtin_amdgcn_readfirstlane((unsigned)(b >> 32)) & 0xffffu,
                       (unsigned)__builtin_amdgcn_readfirstlane(n), 0x00020000u};
        const unsigned lds = (unsigned)(uintptr_t)(__attribute__((address_space(3))) const void*)tile;
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
#pragma unroll
        for (int k = 0; k < COUNT; ++k) {
            const int q = wave + NW * k;
            if (INSTR % NW == 0 || q < INSTR)
                __asm__ volatile("s_mov_b32 m0, %2\n\t"
                                 "s_nop 4\n\t"
                                 "buffer_load_dwordx4 %0, %1, 0 offen lds"
                                 :: "v"(off[k]), "s"(r), "s"(lds + q * 1024) : "memory", "m0");
        }
#pragma clang diagnostic pop
    }
};
// Every direct load of this wave has arrived.
__device__ __forceinline__ void wait_dma() { __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// A barrier that waits for nothing but the waves.
__device__ __forceinline__ void meet() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// both halves of a wave: the larger, the sum
__device__ __forceinline__ float both_max(float x) {
    const u2v r = bits<u2v>(__builtin_amdgcn_permlane32_swap(bits<unsigned>(x), bits<unsigned>(x),
                                                             false, false));
    return fmaxf(bits<float>(r.x), bits<float>(r.y));
}
__device__ __forceinline__ float both_sum(float x) {
    const u2v r = bits<u2v>(__builtin_amdgcn_permlane32_swap(bits<unsigned>(x), bits<unsigned>(x),
                                                             false, false));
    return bits<float>(r.x) + bits<float>(r.y);
}

// Half precision has 5 bits of exponent.  What is rounded to it between two products is
// scaled by powers of two, which change no bit of it in range and are undone in 32 bits:
// probabilities by 2^FORWARD_SHIFT in the forward (at most 1 there) and 2^BACKWARD_SHIFT in
// the backward; dS by 2^DS_SHIFT over the power of two at the largest gradient of the row
// or head.  Without it keys of small probability lose bits to subnormal numbers, and
// gradients of small magnitude vanish.  The other end of the range: dS is finite up to 2^14
// times that power of two, which takes values of several hundred in step with the gradients
// over all of 128 features.
template <class T> constexpr bool NARROW = __is_same(T, _Float16);
template <class T> constexpr int FORWARD_SHIFT = NARROW<T> ? 7 : 0;
template <class T> constexpr int BACKWARD_SHIFT = NARROW<T> ? 12 : 0;
template <class T> constexpr int DS_SHIFT = NARROW<T> ? 2 : 0;

// a score less its row's reference, shifted for the forward.  The difference comes first: taken
// off the reference, the shift would be rounded away beside a bias of the size of 2^24 and more.
template <class T> __device__ __forceinline__ float shifted(float d) {
    return FORWARD_SHIFT<T> ? d + FORWARD_SHIFT<T> : d;
}

// 2^n, n from -126 to 127
__device__ __forceinline__ float pow2(int n) { return bits<float>((unsigned)(127 + n) << 23); }
// the least e with |x| < 2^e; -100 for zero, 0 for infinity and NaN
__device__ __forceinline__ int exponent(float x) {
    const int e = (bits<unsigned>(x) >> 23) & 255;
    return e == 0 ? -100 : e == 255 ? 0 : e - 126;
}

// The wave of a thread, which the compiler must take for the same in all its lanes.
__device__ __forceinline__ int wave_of(int tid) { return __builtin_amdgcn_readfirstlane(tid >> 6); }

// x, which the compiler must take for new in turn n of a loop: what is computed from it is
// computed there, in place of a register (or a spill) for each address.
__device__ __forceinline__ int fresh(int x, int n) {
    __asm__("" : "+v"(x) : "s"(n));
    return x;
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }

// ---------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------
// Philox4x32 with 7 rounds (J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011: the fewest that passed all of BigCrush) on the
// counter (c0, c1, c2, 0).  One draw is a 4 x 4 block of pairs: word i % 4, byte j % 4.
__device__ __forceinline__ u4v philox(unsigned c0, unsigned c1, unsigned c2, unsigned k0,
                                      unsigned k1) {
    unsigned c3 = 0;
#pragma unroll
    for (int r = 0; r < 7; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (unsigned)(b >> 32) ^ c1 ^ k0;
        c2 = (unsigned)(a >> 32) ^ c3 ^ k1;
        c1 = (unsigned)b;
        c3 = (unsigned)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u4v{c0, c1, c2, c3};
}

// w of lane a of four neighbouring lanes: row a of a 4 x 4 matrix, transposed over them
__device__ __forceinline__ u4v quad_transpose(u4v w, int lane) {
    const bool odd = lane & 1, high = lane & 2;
    unsigned t0 = odd ? w.x : w.y, t1 = odd ? w.z : w.w;
    t0 = __builtin_amdgcn_mov_dpp(t0, 0xB1, 0xf, 0xf, true);    // lane ^ 1
    t1 = __builtin_amdgcn_mov_dpp(t1, 0xB1, 0xf, 0xf, true);
    if (odd) { w.x = t0; w.z = t1; } else { w.y = t0; w.w = t1; }
    t0 = high ? w.x : w.z;
    t1 = high ? w.y : w.w;
    t0 = __builtin_amdgcn_mov_dpp(t0, 0x4E, 0xf, 0xf, true);    // lane ^ 2
    t1 = __builtin_amdgcn_mov_dpp(t1, 0x4E, 0xf, 0xf, true);
    if (high) { w.x = t0; w.y = t1; } else { w.z = t0; w.w = t1; }
    return w;
}

struct Drop {
    unsigned k0, k1, c2, least;   // key, batch and head, the least byte that is kept
    float scale;                  // of what is kept

    __device__ __forceinline__ Drop(const d2p_attention_params& p, int bh) {
        unsigned long long s = p.seed;
        if (p.seed_ptr) s = (unsigned long long)*p.seed_ptr;
        k0 = __builtin_amdgcn_readfirstlane((unsigned)s);
        k1 = __builtin_amdgcn_readfirstlane((unsigned)(s >> 32));
        c2 = bh;
        least = p.drop;
        scale = 256.0f / (256 - p.drop);
    }
    // Lane = query i0 + l % 32, accumulators = keys from j0 (i0, j0 multiples of 32): byte
    // v % 4 of word v / 4 is accumulator v's.  The four lanes of a block row draw one of
    // their four blocks each.
    __device__ __forceinline__ u4v by_query(int i0, int j0, int lane) const {
        const u4v w = philox((unsigned)(j0 >> 2) + 2 * (lane & 3) + (lane >> 5),
                             (unsigned)(i0 >> 2) + ((lane & 31) >> 2), c2, k0, k1);
        return quad_transpose(w, lane);
    }
    // Lane = key j0 + l % 32, accumulators = queries from i0; as above.
    __device__ __forceinline__ u4v by_key(int i0, int j0, int lane) const {
        const u4v w = philox((unsigned)(j0 >> 2) + ((lane & 31) >> 2),
                             (unsigned)(i0 >> 2) + 2 * (lane & 3) + (lane >> 5), c2, k0, k1);
        // bytes of one column together: column c of the block in word c
        const unsigned a = __builtin_amdgcn_perm(w.y, w.x, 0x05010400u);   // x0 y0 x1 y1
        const unsigned b = __builtin_amdgcn_perm(w.y, w.x, 0x07030602u);   // x2 y2 x3 y3
        const unsigned c = __builtin_amdgcn_perm(w.w, w.z, 0x05010400u);
        const unsigned d = __builtin_amdgcn_perm(w.w, w.z, 0x07030602u);
        const u4v t = {__builtin_amdgcn_perm(c, a, 0x05040100u),
                       __builtin_amdgcn_perm(c, a, 0x07060302u),
                       __builtin_amdgcn_perm(d, b, 0x05040100u),
                       __builtin_amdgcn_perm(d, b, 0x07060302u)};
        return quad_transpose(t, lane);
    }
    __device__ __forceinline__ bool keeps(u4v w, int v) const {
        return ((w[v >> 2] >> (8 * (v & 3))) & 255u) >= least;
    }
    // Zeros for what is dropped of accumulators 8 f .. 8 f + 7 packed to 16 bits.  All four
    // bytes of a word at once: with t's low seven bits taken off each byte under a borrow-proof
    // top bit, u, a byte is kept if its own top bit and u's agree with t's top bit to that end
    // (their majority with it); a byte permute spreads those bits over the packed halves.
    __device__ __forceinline__ u4v keep16(u4v packed, u4v w, int f) const {
        const unsigned top = 0x80808080u, low = (least & 127u) * 0x01010101u;
        const unsigned less = least & 128u ? 0u : ~0u;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const unsigned x = w[2 * f + n], u = (x | top) - low;
            const unsigned k = (x & u) | ((x | u) & less);
            // selectors 8 and 9: copies of the top bits of bytes 1 and 3; 10 and 11: of
            // bytes 0 and 2, moved up
            packed[2 * n] &= __builtin_amdgcn_perm(k << 8, k, 0x08080a0au);
            packed[2 * n + 1] &= __builtin_amdgcn_perm(k << 8, k, 0x09090b0bu);
        }
        return packed;
    }
};

// ---------------------------------------------------------------------------
// one element of the batch
// ---------------------------------------------------------------------------
struct Span {
    int nq, nk, off;   // lengths; a query's place among the keys is its index + off
    bool bad;          // lengths out of range: the outputs are NaN
    __device__ __forceinline__ Span(const d2p_attention_params& p, int b) {
        nq = p.Lq;
        nk = p.Lk;
        if (p.lengths) {
            nq = p.lengths[2 * b];
            nk = p.lengths[2 * b + 1];
        }
        bad = nq < 0 || nq > p.Lq || nk < 0 || nk > p.Lk;
        if (bad) nq = nk = 0;
        off = p.causal ? nk - nq : 0;
    }
    // the keys that queries up to i see: 0 .. limit - 1
    __device__ __forceinline__ int limit(const d2p_attention_params& p, int i) const {
        return p.causal ? max(min(nk, i + off + 1), 0) : nk;
    }
};

template <class T>
__device__ __forceinline__ Rows head_rows(const void* x, const d2p_strides& s, int b, int h,
                                          int rows, int D) {
    const long long z = (long long)sizeof(T);
    return Rows{(const char*)x + (b * s.batch + h * s.head) * z, s.row * z, rows,
                D / Elem<T>::PER};
}

// A bias in units of log2; a finite one stays finite.
__device__ __forceinline__ float in_log2(float v) {
    const float big = 3.4028235e38f;
    return v >= -big && v <= big ? fminf(fmaxf(v * LOG2E, -big), big) : v;
}

// The bias of each clipped distance for head h, in units of log2: bias[0 .. 2 R] in LDS.
// -inf masks a pair.
template <class T>
__device__ __forceinline__ void load_bias(float* lds, const d2p_attention_params& p, int h,
                                          int tid, int threads) {
    for (int t = tid; t <= 2 * p.max_distance; t += threads) {
        const int n = p.buckets[t];
        float v = __builtin_nanf("");
        if (n >= 0 && n < p.num_buckets) {
            const long long i = (long long)n * p.Hq + h;
            v = p.bias_dtype == D2P_FLOAT32 ? ((const float*)p.bias)[i] : Elem<T>::load(p.bias, i);
            v = in_log2(v);
        }
        lds[t] = v;
    }
}

// Workgroup w of n, handed out so that neighbours run on one XCD (workgroups go round the
// eight XCDs in turn) and share its L2.
__device__ __forceinline__ unsigned near_xcd(unsigned w, unsigned n) {
    const unsigned x = w & 7, q = n >> 3, r = n & 7;
    return x * q + (x < r ? x : r) + (w >> 3);
}

// Head (of all heads of the batch) and block of workgroup w.  An XCD takes whole heads, so
// that their blocks share its L2.  Blocks of equal work go head by head; where work falls
// with the block (`falling`: causal order), an XCD goes through the heaviest blocks of all
// its heads first, and the light ones fill the end.
__device__ __forceinline__ void place(unsigned w, int heads, int blocks, bool falling, int* head,
                                      int* block) {
    const unsigned x = near_xcd(w, (unsigned)heads * blocks);
    *head = x / blocks;
    *block = x % blocks;
    if (falling && heads % 8 == 0) {
        const unsigned own = heads / 8, n = w >> 3;   // of this XCD: its heads, its n-th turn
        *head = (w & 7) * own + n % own;
        *block = n / own;
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline int type_bytes(int dtype) { return dtype == D2P_FLOAT32 ? 4 : 2; }
// Features that the kernels for D work with; 96 with 16 bits only, where it leaves registers
// ([4, 1023, 12 over 3, 80] half with dropout, forward and backward kernels: 168 -> 150 us).
inline int padded(int D, int dtype) {
    return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 && type_bytes(dtype) == 2 ? 96 : 128;
}
__host__ __device__ inline int cdiv(int a, int b) { return (int)(((long long)a + b - 1) / b); }

// Lets `kernel` have up to a compute unit's LDS on the current device; asked for once for
// each kernel and device (`known`: the kernel's own, zeros at first).
struct LdsAllowed {
    std::atomic<bool> on[64];
};
inline int allow_lds(const void* kernel, LdsAllowed& known) {
    int dev = 0;
    D2P_HIP(hipGetDevice(&dev));
    const bool keep = dev >= 0 && dev < 64;
    if (keep && known.on[dev].load(std::memory_order_relaxed)) return D2P_OK;
    D2P_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    if (keep) known.on[dev].store(true, std::memory_order_relaxed);
    return D2P_OK;
}

}  // namespace enc
}  // namespace d2p_amd
