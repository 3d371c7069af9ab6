// Shared pieces of the packed attention kernels (packed_attn.hip, packed_attn_bwd.hip): matrix fragments, LDS tiles, the map from workgroups
// to tiles of sequences, visibility.
//
// One matrix shape throughout, v_mfma_f32_32x32x16: D[32][32] += A[32][16] B[16][32].  Lane l = 32 h + r holds, as A, row r and as B, column r of
// the contraction indices 8 h .. 8 h + 7 (eight 16-bit elements, one ds_read_b128); of D it holds column r and the rows 8 (i / 4) + 4 h + i % 4,
// i = 0..15.  fp32 operands use the same distribution: eight v_mfma_f32_32x32x2_f32, the e-th on element e of every lane.
// A product's result becomes the next product's B operand without leaving its lanes: the rows of D that a lane holds are contraction
// indices then, and any order of them will do as long as A is read in the same one.  So scores are computed transposed (keys x rows): a
// lane owns one query row, its maximum and sum are in-lane but for one exchange between the halves, and the probabilities feed the second
// product from registers.  The A operand of that product is a tile transposed (head columns x keys), which ds_read_b64_tr_b16 reads from the
// row-major tile: four consecutive rows of one column per lane and instruction.
#pragma once
#include "token_types.hpp"

namespace casmtr {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef u32x4 __attribute__((aligned(2))) u32x4_any;   // 16 bytes at any element

// x3_t: fp32 data multiplied as three bf16 terms, x = x0 + x1 + x2 (8 bits each: the 24 bits of x), of whose nine products the six largest are
// kept: what is dropped is below 2^-24 of the product, as the rounding of an fp32 product is.  Six bf16 matrix instructions of 32 cycles
// stand for eight fp32 ones of 64.  Magnitudes from 2^128 (1 - 2^-9) on round to an infinite x0; the products are not finite then, and the careful pass
// (mma_any, mma_hidden) splits them the other way: x0 the largest bf16.
struct x3_t {};
template <typename T> struct FragOf { typedef T type __attribute__((ext_vector_type(8))); };
template <> struct FragOf<x3_t> { struct type { FragOf<bf16_t>::type t[3]; }; };
template <typename T> using frag_t = typename FragOf<T>::type;
template <typename T> struct StoreOf { typedef T type; };   // the type in memory
template <> struct StoreOf<x3_t> { typedef float type; };
template <typename T> using store_t = typename StoreOf<T>::type;

__device__ __forceinline__ f32x16 mma(const frag_t<bf16_t>& a, const frag_t<bf16_t>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const frag_t<f16_t>& a, const frag_t<f16_t>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(const frag_t<float>& a, const frag_t<float>& b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ f32x16 mma(const frag_t<x3_t>& a, const frag_t<x3_t>& b, f32x16 c) {   // the small products first
    c = mma(a.t[2], b.t[0], c);
    c = mma(a.t[0], b.t[2], c);
    c = mma(a.t[1], b.t[1], c);
    c = mma(a.t[1], b.t[0], c);
    c = mma(a.t[0], b.t[1], c);
    return mma(a.t[0], b.t[0], c);
}
// eight values in three terms, two at a time: one conversion to a packed pair, whose halves are the pair's values in fp32 with a shift and a mask
// (11 instructions per pair; from single conversions the compiler makes 15).  CAREFUL: the first term of a finite value is finite
template <bool CAREFUL = false>
__device__ __forceinline__ frag_t<x3_t> split3(const float (&x)[8]) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
    unsigned w[3][4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float u = x[2 * e], v = x[2 * e + 1];
#pragma unroll
        for (int j = 0; j < 3; ++j) {
            f32x2 t = {u, v};
            if constexpr (CAREFUL) {
                const float top = __uint_as_float(0x7f7f0000u);   // the largest bf16
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (__builtin_fabsf(t[i]) < INFINITY) t[i] = __builtin_amdgcn_fmed3f(t[i], -top, top);
            }
            const bf16x2 p = __builtin_convertvector(t, bf16x2);
            __builtin_memcpy(&w[j][e], &p, 4);
            u -= __uint_as_float(w[j][e] << 16);
            v -= __uint_as_float(w[j][e] & 0xffff0000u);
        }
    }
    frag_t<x3_t> f;
    __builtin_memcpy(&f, w, sizeof(f));
    return f;
}
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// An LDS tile of ROWS x DP elements in 16-byte chunks.  Rows are read at one chunk by 32 lanes (ds_read_b128) and, transposed, four rows x four
// chunks by 32 lanes (16-bit) or two rows x eight chunks by 64 lanes (fp32); the exclusive-or below puts the chunks of each such access on
// different banks (256 bytes = all 64 banks = one "line" of 16 chunks; rows shorter than that share a line).
template <typename T, int DP, int ROWS>
struct Tile {
    static constexpr int EPC = 16 / (int)sizeof(T);          // elements of a chunk
    static constexpr int CPR = DP / EPC;                     // chunks of a row
    static constexpr int RB = DP * (int)sizeof(T);           // bytes of a row
    static __device__ __forceinline__ int off(int row, int chunk) {
        if constexpr (CPR >= 16) {
            const int f = sizeof(T) == 2 ? ((row & 3) << 2) | ((row >> 2) & 3) : (((row >> 2) & 1) << 3) | ((row & 3) << 1) | ((row >> 3) & 1);
            return row * RB + ((chunk ^ f) << 4);
        } else if constexpr (CPR == 8) {
            const int line = row >> 1;
            const int f = sizeof(T) == 2 ? ((line & 1) << 2) | ((line >> 1) & 3) : (((line >> 1) & 1) << 3) | (line & 7);
            return line * 256 + (((((row & 1) << 3) | chunk) ^ f) << 4);
        } else {
            const int line = row >> 2;
            return line * 256 + (((((row & 3) << 2) | chunk) ^ (line & 3)) << 4);
        }
    }
    // the (row, chunk) that lies at 16-byte slot p of the tile
    static __device__ __forceinline__ void at(int p, int& row, int& chunk) {
        if constexpr (CPR >= 16) {
            row = p / CPR;
            chunk = (off(row, p % CPR) - row * RB) >> 4;   // (the exclusive-or is its own inverse)
        } else if constexpr (CPR == 8) {
            const int line = p >> 4, x = ((off(2 * line, 0) - line * 256) >> 4) ^ (p & 15);
            row = 2 * line + (x >> 3);
            chunk = x & 7;
        } else {
            const int line = p >> 4, x = (line & 3) ^ (p & 15);
            row = 4 * line + (x >> 2);
            chunk = x & 3;
        }
    }
    // A / B operand: row `row` (per lane), contraction indices 16 s + 8 h ..
    static __device__ __forceinline__ frag_t<T> rows(const char* tile, int row, int s, int h) {
        frag_t<T> f;
        if constexpr (sizeof(T) == 2) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(tile + off(row, 2 * s + h));
            __builtin_memcpy(&f, &v, 16);
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4*>(tile + off(row, 4 * s + 2 * h));
            const f32x4 b = *reinterpret_cast<const f32x4*>(tile + off(row, 4 * s + 2 * h + 1));
#pragma unroll
            for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
        }
        return f;
    }
    // transposed A operand: column col0 + r of the tile's rows row0 + 4 h + {0..3} and row0 + 8 + 4 h + {0..3} -- the order in which a result's
    // registers 8 t .. 8 t + 7 hold its rows
    static __device__ __forceinline__ frag_t<T> cols(const char* tile, int row0, int col0, int lane) {
        frag_t<T> f;
        const int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // the 16 lanes of a group name four rows x 16 columns (8 bytes each); lane i receives column i of the four rows
            const int i = lane & 15, row = row0 + 4 * h + (i >> 2), col = col0 + (lane & 16) + 4 * (i & 3);
            const int half = (col & 4) << 1;
            typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + off(row, col >> 3) + half));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(tile + off(row + 8, col >> 3) + half));
            __builtin_memcpy(&f, &a, 8);
            __builtin_memcpy(reinterpret_cast<char*>(&f) + 8, &b, 8);
        } else {
            const int col = col0 + (lane & 31);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                f[e] = *reinterpret_cast<const float*>(tile + off(row0 + 8 * (e >> 2) + 4 * h + (e & 3), col >> 2) + (col & 3) * 4);
        }
        return f;
    }
};

// x3_t: one tile per term, one behind the other
template <int DP, int ROWS>
struct Tile<x3_t, DP, ROWS> {
    typedef Tile<bf16_t, DP, ROWS> P;
    static constexpr int RB = 3 * P::RB, PLANE = ROWS * P::RB;
    static __device__ __forceinline__ frag_t<x3_t> rows(const char* tile, int row, int s, int h) {
        return {{P::rows(tile, row, s, h), P::rows(tile + PLANE, row, s, h), P::rows(tile + 2 * PLANE, row, s, h)}};
    }
    static __device__ __forceinline__ frag_t<x3_t> cols(const char* tile, int row0, int col0, int lane) {
        return {{P::cols(tile, row0, col0, lane), P::cols(tile + PLANE, row0, col0, lane), P::cols(tile + 2 * PLANE, row0, col0, lane)}};
    }
};

// 16 bytes of a row from column col on; columns from D on are zero
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int col, int D) {
    constexpr int EPC = 16 / (int)sizeof(T);
    if (col + EPC <= D) return *reinterpret_cast<const u32x4_any*>(row + col);
    T v[EPC];
#pragma unroll
    for (int i = 0; i < EPC; ++i) v[i] = col + i < D ? row[col + i] : (T)0.f;
    u32x4 r;
    __builtin_memcpy(&r, v, 16);
    return r;
}
// the fragment of a row held in global memory: columns 16 s + 8 h ..
template <typename T, bool CAREFUL = false>
__device__ __forceinline__ frag_t<T> load_frag(const store_t<T>* row, int s, int h, int D) {
    frag_t<T> f;
    const int col = 16 * s + 8 * h;
    if constexpr (std::is_same<T, x3_t>::value) {
        float x[8];
        const u32x4 a = load_chunk(row, col, D), b = load_chunk(row, col + 4, D);
        __builtin_memcpy(x, &a, 16);
        __builtin_memcpy(x + 4, &b, 16);
        f = split3<CAREFUL>(x);
    } else {
        const u32x4 a = load_chunk(row, col, D);
        __builtin_memcpy(&f, &a, 16);
        if constexpr (sizeof(T) == 4) {
            const u32x4 b = load_chunk(row, col + 4, D);
            __builtin_memcpy(reinterpret_cast<char*>(&f) + 16, &b, 16);
        }
    }
    return f;
}

// ---- a tile straight from global memory into LDS (buffer_load_dwordx4 ... lds: 64 lanes x 16 bytes to consecutive LDS addresses, no
// registers; the layout's exclusive-or is applied to the SOURCE addresses).  The buffer's size is set per tile to the rows that are left, and
// what lies behind it -- rows past the sequence's keys, columns past D -- arrives as zero.  Needs 16-byte aligned rows of whole chunks that do not
// overlap.  Inline asm, so that the compiler does not drain the loads in flight before every LDS read: the kernels wait with glds_wait().
template <typename T, int DP, int ROWS, int NW>
struct TileDma {
    typedef Tile<T, DP, ROWS> L;
    static constexpr int N = ROWS * L::CPR / (64 * NW);   // instructions per wave
    unsigned voff[N];
    unsigned row_bytes, width;
    __device__ __forceinline__ void init(int tid, long long stride, int D) {
        row_bytes = (unsigned)(stride * (long long)sizeof(T));
        width = (unsigned)(D * (int)sizeof(T));
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int row, chunk;
            L::at(tid + 64 * NW * i, row, chunk);
            voff[i] = chunk * L::EPC < D ? (unsigned)row * row_bytes + (unsigned)chunk * 16u : 0x80000000u;
        }
    }
    // rows_left >= 1 rows from `base` on; lds: the tile's LDS byte address
    __device__ __forceinline__ void issue(const T* base, int rows_left, unsigned lds, int wave) const {
        const unsigned long long b = (unsigned long long)base;
        const u32x4 rsrc = {(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)b), (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(b >> 32)),
                            (unsigned)__builtin_amdgcn_readfirstlane((int)((unsigned)(min(rows_left, ROWS) - 1) * row_bytes + width)), 0x00020000u};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const unsigned dst = (unsigned)__builtin_amdgcn_readfirstlane((int)(lds + (unsigned)(64 * NW * i + 64 * wave) * 16u));
            asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %2, 0 offen lds" ::"v"(voff[i]), "s"(dst), "s"(rsrc) : "memory", "m0");
        }
    }
    // whether rows of this stride can be read so
    static __host__ __forceinline__ bool fits(const void* p, long long token_stride, long long head_stride, int D) {
        const long long e = (long long)sizeof(T);
        return D * e % 16 == 0 && (unsigned long long)p % 16 == 0 && token_stride * e % 16 == 0 && head_stride * e % 16 == 0 && token_stride >= D &&
               token_stride * e * (ROWS + 1) < 0x7fffffffLL;
    }
};

// Two tiles of ROWS x DP in two stages of LDS (K and V, or q and the output's gradient): rows t ROWS .. of `a` and `b`, zero from `count` rows and D
// columns on.  fetch(t, stage) starts tile t, arrived(stage) is called by every thread before the barrier that precedes its use.
// DMA: straight into LDS; otherwise (rows that are not 16-byte aligned) through registers, written when the tile is due.
template <typename T, int DP, int ROWS, int NW, bool DMA>
struct TilePair {
    typedef Tile<T, DP, ROWS> L;
    static constexpr int NT = 64 * NW, NCH = ROWS * L::CPR / NT, TB = ROWS * L::RB, BYTES = 4 * TB;
    static_assert(ROWS * L::CPR % NT == 0, "whole chunks per thread");
    char* smem;
    const T *a, *b;
    long long as, bs;
    int count, D, tid, wave;
    TileDma<T, DP, ROWS, NW> ad, bd;
    u32x4 ar[DMA ? 1 : NCH], br[DMA ? 1 : NCH];
    __device__ __forceinline__ void init(char* smem_, int tid_, int wave_, long long as_, long long bs_, int D_) {
        smem = smem_; tid = tid_; wave = wave_; as = as_; bs = bs_; D = D_;
        if constexpr (DMA) { ad.init(tid, as, D); bd.init(tid, bs, D); }
    }
    __device__ __forceinline__ void of(const T* a_, const T* b_, int count_) { a = a_; b = b_; count = count_; }
    __device__ __forceinline__ const char* first(int stage) const { return smem + 2 * stage * TB; }
    __device__ __forceinline__ const char* second(int stage) const { return smem + (2 * stage + 1) * TB; }
    __device__ __forceinline__ void fetch(int t, int stage) {
        if constexpr (DMA) {
            const unsigned lds = lds_byte_addr(smem) + 2 * stage * TB;
            ad.issue(a + (long long)t * ROWS * as, count - t * ROWS, lds, wave);
            bd.issue(b + (long long)t * ROWS * bs, count - t * ROWS, lds + TB, wave);
        } else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int id = tid + NT * i, rr = t * ROWS + id / L::CPR, c = (id % L::CPR) * L::EPC;
                ar[i] = u32x4{0, 0, 0, 0};
                br[i] = u32x4{0, 0, 0, 0};
                if (rr < count && c < D) {
                    ar[i] = load_chunk(a + (long long)rr * as, c, D);
                    br[i] = load_chunk(b + (long long)rr * bs, c, D);
                }
            }
        }
    }
    template <bool CAREFUL = false>
    __device__ __forceinline__ void arrived(int stage) {
        if constexpr (DMA) glds_wait<0>();
        else {
#pragma unroll
            for (int i = 0; i < NCH; ++i) {
                const int id = tid + NT * i, o = L::off(id / L::CPR, id % L::CPR);
                *reinterpret_cast<u32x4*>(smem + 2 * stage * TB + o) = ar[i];
                *reinterpret_cast<u32x4*>(smem + (2 * stage + 1) * TB + o) = br[i];
            }
        }
    }
};

// x3_t: fp32 rows through registers, split on the way into LDS
template <int DP, int ROWS, int NW>
struct TilePair<x3_t, DP, ROWS, NW, false> {
    typedef Tile<x3_t, DP, ROWS> L;
    typedef Tile<bf16_t, DP, ROWS> P;
    static constexpr int NT = 64 * NW, N = ROWS * P::CPR / NT, TB = 3 * L::PLANE, BYTES = 4 * TB;
    static_assert(ROWS * P::CPR % NT == 0, "whole chunks per thread");
    char* smem;
    const float *a, *b;
    long long as, bs;
    int count, D, tid;
    u32x4 ar[2 * N], br[2 * N];
    __device__ __forceinline__ void init(char* smem_, int tid_, int, long long as_, long long bs_, int D_) { smem = smem_; tid = tid_; as = as_; bs = bs_; D = D_; }
    __device__ __forceinline__ void of(const float* a_, const float* b_, int count_) { a = a_; b = b_; count = count_; }
    __device__ __forceinline__ const char* first(int stage) const { return smem + 2 * stage * TB; }
    __device__ __forceinline__ const char* second(int stage) const { return smem + (2 * stage + 1) * TB; }
    __device__ __forceinline__ void fetch(int t, int) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = tid + NT * i, rr = t * ROWS + id / P::CPR, c = (id % P::CPR) * 8;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                ar[2 * i + j] = u32x4{0, 0, 0, 0};
                br[2 * i + j] = u32x4{0, 0, 0, 0};
                if (rr < count && c + 4 * j < D) {
                    ar[2 * i + j] = load_chunk(a + (long long)rr * as, c + 4 * j, D);
                    br[2 * i + j] = load_chunk(b + (long long)rr * bs, c + 4 * j, D);
                }
            }
        }
    }
    template <bool CAREFUL>
    static __device__ __forceinline__ void put(char* tile, int o, const u32x4& lo, const u32x4& hi) {
        float x[8];
        __builtin_memcpy(x, &lo, 16);
        __builtin_memcpy(x + 4, &hi, 16);
        const frag_t<x3_t> f = split3<CAREFUL>(x);
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<frag_t<bf16_t>*>(tile + j * L::PLANE + o) = f.t[j];
    }
    template <bool CAREFUL = false>
    __device__ __forceinline__ void arrived(int stage) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = tid + NT * i, o = P::off(id / P::CPR, id % P::CPR);
            put<CAREFUL>(smem + 2 * stage * TB, o, ar[2 * i], ar[2 * i + 1]);
            put<CAREFUL>(smem + (2 * stage + 1) * TB, o, br[2 * i], br[2 * i + 1]);
        }
    }
};

// registers 8 t .. 8 t + 7 of a result as the next product's operand
template <typename T>
__device__ __forceinline__ frag_t<T> to_frag(const f32x16& c, int t) {
    if constexpr (std::is_same<T, x3_t>::value) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = c[8 * t + e];
        return split3(x);
    } else {
        frag_t<T> f;
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] = (T)c[8 * t + e];
        return f;
    }
}

__device__ __forceinline__ float max_halves(float v) {   // max / sum with the other half of the wave
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float add_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// `v` where x < limit, `hidden` elsewhere.  In bits, not as `if` or `?:`: those become control flow that the compiler merges with the wave-uniform
// `if` around the masks, and then every tile pays for them.
__device__ __forceinline__ float seen_or(float v, float hidden, int x, int limit) {
    const unsigned m = (unsigned)((x - limit) >> 31);
    return __uint_as_float((__float_as_uint(v) & m) | (__float_as_uint(hidden) & ~m));
}

// whether any of the wave's eight elements is infinite or NaN
template <typename T>
__device__ __forceinline__ bool any_not_finite(const frag_t<T>& f) {
    constexpr unsigned EXP = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, bf16_t>::value ? 0x7f807f80u : 0x7c007c00u;
    constexpr unsigned ONE = sizeof(T) == 4 ? 0x00800000u : std::is_same<T, bf16_t>::value ? 0x00800080u : 0x04000400u;
    constexpr unsigned TOP = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    unsigned w[sizeof(frag_t<T>) / 4], acc = 0;
    __builtin_memcpy(w, &f, sizeof(w));
#pragma unroll
    for (unsigned i = 0; i < sizeof(w) / 4; ++i) acc |= (w[i] & EXP) + ONE;   // an exponent of all ones carries into the sign's place
    return __any((acc & TOP) != 0);
}
// c += A B where some (contraction index, column) pairs are hidden: B is zero there, and what A holds at an index must not reach the columns
// that it is hidden from, infinities and NaN included (0 * inf is NaN).  If A is finite that is the plain product; otherwise its finite
// elements are multiplied first and the others follow index by index, a column taking the sum only where it sees the index: every
// column gets the bits that it would get without them.  sees(n): whether this lane's column sees the index that element n & 7 of
// half n >> 3 stands for.
template <typename T, typename Sees>
__device__ __forceinline__ f32x16 mma_hidden(const frag_t<T>& a, const frag_t<T>& b, f32x16 c, int h, Sees&& sees) {
    constexpr bool X3 = std::is_same<T, x3_t>::value;
    const auto& a0 = [&]() -> const auto& { if constexpr (X3) return a.t[0]; else return a; }();   // (of the terms, the first says it)
    typedef std::conditional_t<X3, bf16_t, T> E;
    if (__builtin_expect(!any_not_finite<E>(a0), 1)) return mma(a, b, c);
    frag_t<T> fin;
    unsigned odd = 0;   // this lane's elements that are not finite
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool ok = __builtin_fabsf((float)a0[e]) < INFINITY;
        if constexpr (X3) {
#pragma unroll
            for (int j = 0; j < 3; ++j) fin.t[j][e] = ok ? a.t[j][e] : (E)0.f;
        } else fin[e] = ok ? a[e] : (E)0.f;
        odd |= (ok ? 0u : 1u) << (8 * h + e);
    }
    c = mma(fin, b, c);
    for (int n = 0; n < 16; ++n) {
        if (!__any((odd >> n) & 1u)) continue;
        frag_t<E> a1, b1;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool on = n == 8 * h + e;
            a1[e] = on && ((odd >> n) & 1u) ? a0[e] : (E)0.f;
            if constexpr (X3) b1[e] = on ? b.t[0][e] : (E)0.f;
            else b1[e] = on ? b[e] : (E)0.f;
        }
        const f32x16 d = mma(a1, b1, c);
        if (sees(n)) c = d;
    }
    return c;
}
// c += A B as the formula has it where either holds infinities or NaN.  Of three terms the second and third of an infinity are NaN: such elements
// are left out of the product of terms (so that the other pairs keep its bits), and an index that has any is multiplied by itself, first
// terms only: what is not finite then is what the left-out elements add.
template <typename T>
__device__ __forceinline__ f32x16 mma_any(const frag_t<T>& a, const frag_t<T>& b, f32x16 c, int h) {
    if constexpr (!std::is_same<T, x3_t>::value) return mma(a, b, c);
    else {
        if (!any_not_finite<bf16_t>(a.t[0]) && !any_not_finite<bf16_t>(b.t[0])) return mma(a, b, c);
        frag_t<x3_t> fa, fb;
        unsigned odd = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool ka = __builtin_fabsf((float)a.t[0][e]) < INFINITY, kb = __builtin_fabsf((float)b.t[0][e]) < INFINITY;
#pragma unroll
            for (int j = 0; j < 3; ++j) {
                fa.t[j][e] = ka ? a.t[j][e] : (bf16_t)0.f;
                fb.t[j][e] = kb ? b.t[j][e] : (bf16_t)0.f;
            }
            odd |= (ka && kb ? 0u : 1u) << (8 * h + e);
        }
        c = mma(fa, fb, c);
        for (int n = 0; n < 16; ++n) {
            if (!__any((odd >> n) & 1u)) continue;
            frag_t<bf16_t> a1, b1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool on = n == 8 * h + e;
                a1[e] = on ? a.t[0][e] : (bf16_t)0.f;
                b1[e] = on ? b.t[0][e] : (bf16_t)0.f;
            }
            const f32x16 d = mma(a1, b1, zero16());
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (!(__builtin_fabsf(d[i]) < INFINITY)) c[i] += d[i];
        }
        return c;
    }
}

// ---- sequences
struct PackedSeqs {
    const int *cu_q, *cu_k, *len_k;   // cu_q, cu_k [n + 1]; len_k [n] or NULL: keys in use of each sequence's share
    int n, G;                         // sequences; query heads per key head
    int causal;
    long long Tq, Tk;
};
struct Span { int begin, count; };
// The rows of "sequence" s = -1 .. n: -1 and n are the rows before the first and behind the last one, which belong to none.  Whatever the
// arrays hold, spans stay inside the tensors.  The loads are unconditional (indices clamped), so that those of a span and of both spans
// of a sequence travel together: a workgroup's first tile waits for three round trips to memory, its place, its spans, its data.
__device__ __forceinline__ int bound_of(const int* cu, int s, int n, long long T) {
    const int v = (int)max(0LL, min((long long)cu[max(0, min(s, n))], T));
    return s < 0 ? 0 : s > n ? (int)T : v;
}
__device__ __forceinline__ Span span_of(const int* cu, int s, int n, long long T) {
    const int b = bound_of(cu, s, n, T), e = bound_of(cu, s + 1, n, T);
    return {b, max(0, e - b)};
}
__device__ __forceinline__ Span keys_of(const PackedSeqs& p, int s) {
    const bool none = s < 0 || s >= p.n;
    Span k = span_of(p.cu_k, s, p.n, p.Tk);
    if (p.len_k) {
        const int used = p.n > 0 ? p.len_k[max(0, min(s, p.n - 1))] : 0;
        k.count = max(0, min(k.count, used));
    }
    return none ? Span{0, 0} : k;
}
// Tiles of SIZE rows (a token counts `per` rows): sequence s owns the slots from bound(s) * per / SIZE + s + 1 on, which leaves it at least
// as many as it has tiles, whatever the lengths.  So the host sizes the grid from the tensors' shapes alone -- it never waits for the
// lengths -- and a workgroup looks its tile up; slots too many leave at once.
__host__ __device__ __forceinline__ long long slot_count(long long T, int per, int n, int size) { return T * per / size + n + 2; }
__device__ __forceinline__ int seq_of_slot(const int* cu, int n, long long T, int per, int size, long long slot, int* tile) {
    // the last s whose first slot is <= slot; 64 candidates at a time, one per lane: one round trip up to 62 sequences, two up to 4000
    const int lane = threadIdx.x & 63;
    const auto first = [&](int s) { return (long long)bound_of(cu, s, n, T) * per / size + s + 1; };
    int lo = -1, hi = n;
    for (;;) {
        const int step = (hi - lo) / 64 + 1;
        const long long s = (long long)lo + (long long)lane * step;
        const unsigned long long below = __ballot(s <= hi && (lane == 0 || first((int)min(s, (long long)hi)) <= slot));   // (lane 0: known)
        lo += (63 - __builtin_clzll(below)) * step;
        hi = (int)min((long long)hi, (long long)lo + step - 1);
        if (step == 1) break;
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    *tile = (int)max(0LL, slot - first(lo));   // (never negative for non-decreasing bounds)
    return lo;
}
}  // namespace casmtr
