// Attention over packed sequences, backward.  With p_ij = exp(scale q_i . k_j - lse_i):
//   delta_i = sum_d do_i o_i;  ds_ij = p_ij (do_i . v_j - delta_i) scale
//   dq_i = sum_j ds_ij k_j;    dk_j = sum_i ds_ij q_i;    dv_j = sum_i p_ij do_i
// No atomics: one kernel owns query rows and walks the keys (dq, and delta on the way), one owns keys and walks the query rows of all
// heads that share them (dk, dv: the sum over the group is in the accumulator; in parts that a third kernel adds where there are few keys).  The scores are computed twice for it -- 7 products
// instead of 5 -- and results repeat bit for bit.  Bound by the matrix instructions and, for heads of 64 and less, the exponentials beside them.
// 16384 causal tokens, bf16: 32 / 8 heads of 128 dq 2.87 ms (1.15 PFLOP/s), dk and dv 5.6 ms (0.78; one wave per SIMD: K, V and both sums take 435
// registers); 16 heads of 64 dq 0.79 ms (1.05), dk and dv 1.12 ms (0.98).
// Roundings to 16 bits: p and ds, for the products with them.  In fp16 at a power of two that keeps them in its normal range: p (at most 1, the smaller
// the more keys there are) at 2^12, ds, whose size follows the gradient's, at a running one (in_range).  Unscaled, gradients of 1e-3 over
// 4096 keys lost most of their bits on the way to dq and dk.  It costs the largest and a product per element: the same sizes in fp16 take dq 3.18, dk and dv
// 5.7 ms; 0.92 and 1.26 ms.
#include "packed_attn.hpp"

using namespace casmtr;

namespace {
struct BwdArgs {
    const void *q, *k, *v, *o, *g;     // o, g (the gradient of o): [Tq, H, D] contiguous
    const float* lse;
    float* delta;                      // [Tq, H]
    float* part;                       // splits > 1: [splits][dk, dv][Tk * Hk * D] partial sums
    void *dq, *dk, *dv;                // contiguous
    PackedSeqs s;
    long long qts, qhs, kts, khs, vts, vhs;
    int H, Hk, D, splits;
    float scale, scale_log2;
};
constexpr float LOG2E = 1.44269504088896341f;

// the four consecutive columns that a lane holds of each 8 columns of a transposed result, to a row in the output's type
template <typename T, int DB>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&acc)[DB], int h, int D, float f) {
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * d + 8 * g + 4 * h;
            typedef T T4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
            T4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(acc[d][4 * g + e] * f);
            if (c + 4 <= D) *reinterpret_cast<T4*>(row + c) = v;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (c + e < D) row[c + e] = v[e];
        }
}

// bits by which p is raised for the product with do.  Not all 15 that there are: lse is rounded, and where scores are so large that this shows, p may
// come out somewhat above 1.
template <typename T> constexpr float P_BITS = std::is_same<T, f16_t>::value ? 12.f : 0.f;
// fp16: x (32 contraction indices of this lane's column) times 2^e, where e brings the column's largest |x| so far to 2^8 at least and below 2^15; when one
// comes that passes that, e is lowered and the sums so far follow, which is exact.  What is rounded below the normal range then loses at most
// 2^-33 of the largest.  (e starts at 127, where the first |x| of 2^-112 or more lowers it.)  Infinities and NaN stay what they are.
constexpr int E_START = 127;
template <typename T, int DB>
__device__ __forceinline__ void in_range(f32x16& x, f32x16 (&sum)[DB], int& e) {
    if constexpr (std::is_same<T, f16_t>::value) {
        float big[4] = {__builtin_fabsf(x[0]), __builtin_fabsf(x[1]), __builtin_fabsf(x[2]), __builtin_fabsf(x[3])};
#pragma unroll
        for (int i = 4; i < 16; ++i) big[i & 3] = fmaxf(big[i & 3], __builtin_fabsf(x[i]));
        const float mx = max_halves(fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])));   // (both halves hold parts of the column's sum)
        const int ex = (int)((__float_as_uint(mx) >> 23) & 255u) - 127;                      // -127 (zero) .. 128 (infinity)
        const bool up = ex + e > 14;
        if (__any(up)) {
            const int lower = up ? 8 - ex - e : 0;
            e += lower;
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[d][i] = __builtin_amdgcn_ldexpf(sum[d][i], lower);
        }
        const float f = __uint_as_float((unsigned)(e + 127) << 23);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= f;
    }
}
// the factor that takes 2^e and `bits` out of such a sum again
template <typename T>
__device__ __forceinline__ float out_of_range(float f, int e, float bits = 0.f) {
    if constexpr (std::is_same<T, f16_t>::value) return __builtin_amdgcn_ldexpf(f, -e - (int)bits);
    else return f;
}

template <int DB>
__device__ __forceinline__ bool not_finite(const f32x16 (&acc)[DB]) {
    float worst = 0.f;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) worst += __builtin_fabsf(acc[d][i]);
    return !(worst < INFINITY);
}

// dq: a workgroup's rows are (token, head) pairs as in the forward kernel
template <typename T, int DP, int BN, int NW, bool DMA>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 || (sizeof(T) == 1 && DP <= 64) ? (sizeof(T) == 2 && DP <= 64 ? 3 : 2) : 1) void packed_attn_dq_kernel(const BwdArgs a) {
    typedef Tile<T, DP, BN> L;
    constexpr int BM = 32 * NW, KS = DP / 16, NB = BN / 32, DB = DP / 32;
    __shared__ __attribute__((aligned(256))) char smem[TilePair<T, DP, BN, NW, DMA>::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, r = lane & 31;
    const int hk = blockIdx.x % a.Hk, G = a.s.G;
    int tile;
    const int seq = seq_of_slot(a.s.cu_q, a.s.n, a.s.Tq, G, BM, (long long)(gridDim.x / a.Hk - 1 - blockIdx.x / a.Hk), &tile);
    const Span rows = span_of(a.s.cu_q, seq, a.s.n, a.s.Tq), keys = keys_of(a.s, seq);
    const int nrow = rows.count * G;
    if ((long long)tile * BM >= nrow) return;
    const int row0 = tile * BM;
    const int row = row0 + 32 * wave + r, rc = min(row, nrow - 1), tok = rc / G, head = hk * G + rc % G;
    const int shift = keys.count - rows.count;
    const auto limit_at = [&](int rr) { return a.s.causal ? max(0, min(keys.count, min(rr, nrow - 1) / G + shift + 1)) : keys.count; };
    const int limit = limit_at(row);
    const int wg_end = limit_at(row0 + BM - 1), wave_end = limit_at(row0 + 32 * wave + 31), wave_all = limit_at(row0 + 32 * wave);
    const int t1 = (wg_end + BN - 1) / BN;
    const long long out_row = (long long)(rows.begin + tok) * a.H + head;
    frag_t<T> qf[KS], gf[KS];
    const auto load_rows = [&](auto guard) {
        const store_t<T>* qr = (const store_t<T>*)a.q + (long long)(rows.begin + tok) * a.qts + head * a.qhs;
        const store_t<T>* gr = (const store_t<T>*)a.g + out_row * a.D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = load_frag<T, decltype(guard)::value>(qr, s, h, a.D);
            gf[s] = load_frag<T, decltype(guard)::value>(gr, s, h, a.D);
        }
    };
    load_rows(std::false_type{});
    float delta = 0.f;
    {
        const store_t<T> *gr = (const store_t<T>*)a.g + out_row * a.D, *orow = (const store_t<T>*)a.o + out_row * a.D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            float x[8], y[8];
            const int c = 16 * s + 8 * h, n = a.D - c;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[e] = 0.f;
            if (n > 0) { load_n(gr + c, x, n); load_n(orow + c, y, n); }
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(x[e], y[e], delta);
        }
    }
    delta = add_halves(delta);
    const float lse = a.lse[out_row], lse2 = lse == -INFINITY ? 0.f : lse * LOG2E;   // (a row that sees nothing: every key is hidden below)
    if (h == 0 && row < nrow) a.delta[out_row] = delta;
    f32x16 acc[DB];
    int e = E_START;
    TilePair<T, DP, BN, NW, DMA> kv;
    kv.init(smem, tid, wave, a.kts, a.vts, a.D);
    kv.of((const store_t<T>*)a.k + (long long)keys.begin * a.kts + hk * a.khs, (const store_t<T>*)a.v + (long long)keys.begin * a.vts + hk * a.vhs, keys.count);
    const auto pass = [&](auto guard) {
        constexpr bool GUARD = decltype(guard)::value;
        e = E_START;
        if (GUARD && std::is_same<T, x3_t>::value) load_rows(guard);
#pragma unroll
        for (int d = 0; d < DB; ++d) acc[d] = zero16();
        if (0 < t1) kv.fetch(0, 0);
        const auto step = [&](int t, auto stage_) {
            constexpr int stage = decltype(stage_)::value;
            kv.template arrived<GUARD>(stage);
            __syncthreads();
            if (t + 1 < t1) kv.fetch(t + 1, stage ^ 1);
            if (t * BN >= wave_end) return;
            const bool hidden = (t + 1) * BN > wave_all;
            const char *ks = kv.first(stage), *vs = kv.second(stage);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    const frag_t<T> kf = L::rows(ks, 32 * b + r, st, h), vf = L::rows(vs, 32 * b + r, st, h);
                    s = GUARD ? mma_any<T>(kf, qf[st], s, h) : mma(kf, qf[st], s);
                    dp = GUARD ? mma_any<T>(vf, gf[st], dp, h) : mma(vf, gf[st], dp);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, -lse2));
                    s[i] = p * (dp[i] - delta);
                }
                if (hidden) {
                    const int lim = limit - t * BN - 4 * h;
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[i] = seen_or(s[i], 0.f, 32 * b + 8 * (i >> 2) + (i & 3), lim);
                }
                in_range<T, DB>(s, acc, e);
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const frag_t<T> ds = to_frag<T>(s, tt);   // rounded to the keys' type for the product with them
                    const int k0 = 32 * b + 16 * tt;
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const frag_t<T> kt = L::cols(ks, k0, 32 * d, lane);
                        if constexpr (!GUARD) acc[d] = mma(kt, ds, acc[d]);
                        else acc[d] = mma_hidden<T>(kt, ds, acc[d], h, [&](int n) { return t * BN + k0 + 8 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3) < limit; });
                    }
                }
            }
        };
        for (int t = 0; t < t1; t += 2) {
            step(t, std::integral_constant<int, 0>{});
            if (t + 1 < t1) step(t + 1, std::integral_constant<int, 1>{});
        }
    };
    pass(std::false_type{});
    if (a.s.causal || std::is_same<T, x3_t>::value) {   // as in the forward kernel: a sum that is not finite may have met a hidden infinity
        if (__syncthreads_or(not_finite(acc))) pass(std::true_type{});
    }
    if (row < nrow) store_row<store_t<T>, DB>((store_t<T>*)a.dq + out_row * a.D, acc, h, a.D, out_of_range<T>(a.scale, e));
}

// dk, dv: a workgroup owns BN = 32 NW keys of one key head, a wave 32 of them (K and V stay in its registers), and walks the rows of the heads that
// share it, head by head in tiles of BM tokens
template <typename T, int DP, int BM, int NW, bool DMA>
__global__ __launch_bounds__(64 * NW, (sizeof(T) == 2 && DP <= 64) || (sizeof(T) == 1 && DP <= 32) ? 2 : 1) void packed_attn_dkv_kernel(const BwdArgs a) {
    typedef Tile<T, DP, BM> L;
    constexpr int BN = 32 * NW, KS = DP / 16, MB = BM / 32, DB = DP / 32;
    static_assert(BM <= 64 * NW, "a thread stages one row's statistics");
    __shared__ __attribute__((aligned(256))) char smem[TilePair<T, DP, BM, NW, DMA>::BYTES];
    __shared__ __attribute__((aligned(16))) float stat[2][2][BM];        // lse (in bits), delta of two stages
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, r = lane & 31;
    const int hk = blockIdx.x % a.Hk, G = a.s.G;
    int tile;
    const int seq = seq_of_slot(a.s.cu_k, a.s.n, a.s.Tk, 1, BN, (long long)(blockIdx.x / a.Hk), &tile);   // earlier keys are seen by more rows: first
    const Span share = span_of(a.s.cu_k, seq, a.s.n, a.s.Tk), keys = keys_of(a.s, seq);
    const Span rows = seq >= 0 && seq < a.s.n ? span_of(a.s.cu_q, seq, a.s.n, a.s.Tq) : Span{0, 0};
    if ((long long)tile * BN >= share.count) return;
    const int key0 = tile * BN, wk = key0 + 32 * wave, key = wk + r;      // keys of the share that are not in use get zero gradients
    const int shift = keys.count - rows.count;
    const bool used = key < keys.count;
    // a key is seen by the tokens from first_of(key) on: of the lane's key, of the first of the wave and of the workgroup, of the wave's last
    const auto first_of = [&](int j) { return j >= keys.count ? rows.count : a.s.causal ? min(rows.count, max(0, j - shift)) : 0; };
    const int first = first_of(key), wg_first = first_of(key0), wave_first = first_of(wk), wave_all = first_of(wk + 31);
    const int kc = max(0, min(key, keys.count - 1));
    frag_t<T> kf[KS], vf[KS];
    const auto load_keys = [&](auto guard) {
        const store_t<T>* kr = (const store_t<T>*)a.k + (long long)(keys.begin + kc) * a.kts + hk * a.khs;
        const store_t<T>* vr = (const store_t<T>*)a.v + (long long)(keys.begin + kc) * a.vts + hk * a.vhs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[s] = load_frag<T, decltype(guard)::value>(kr, s, h, keys.count > 0 ? a.D : 0);
            vf[s] = load_frag<T, decltype(guard)::value>(vr, s, h, keys.count > 0 ? a.D : 0);
        }
    };
    load_keys(std::false_type{});
    f32x16 dk[DB], dv[DB];
    int e = E_START;
    const int t0 = wg_first / BM, per = (rows.count + BM - 1) / BM - t0;   // tiles of a head
    int n0 = 0, turns = wg_first < rows.count ? per * G : 0;                // of all heads, of this split
    if (a.splits > 1) {
        const int each = (turns + a.splits - 1) / a.splits;
        n0 = min(turns, each * (int)blockIdx.y);
        turns = min(turns, n0 + each);
    }
    TilePair<T, DP, BM, NW, DMA> qg;
    qg.init(smem, tid, wave, a.qts, (long long)a.H * a.D, a.D);
    float sl = 0.f, sd = 0.f;
    const auto fetch = [&](int n, int stage) {   // turn n: tile t0 + n % per of the group's head n / per
        const int hd = hk * G + n / per, t = t0 + n % per;
        if (tid < BM) {
            const int tok = t * BM + tid;
            sl = INFINITY;   // a row that sees nothing: its probabilities are exactly 0
            sd = 0.f;
            if (tok < rows.count) {
                const long long at = (long long)(rows.begin + tok) * a.H + hd;
                const float x = a.lse[at];
                sl = x == -INFINITY ? INFINITY : x * LOG2E - P_BITS<T>;
                sd = a.delta[at];
            }
        }
        qg.of((const store_t<T>*)a.q + (long long)rows.begin * a.qts + hd * a.qhs, (const store_t<T>*)a.g + ((long long)rows.begin * a.H + hd) * a.D, rows.count);
        qg.fetch(t, stage);
    };
    const auto pass = [&](auto guard) {
        constexpr bool GUARD = decltype(guard)::value;
#pragma unroll
        for (int d = 0; d < DB; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
        e = E_START;
        if (GUARD && std::is_same<T, x3_t>::value) load_keys(guard);
        if (n0 < turns) fetch(n0, 0);
        const auto step = [&](int n, auto stage_) {
            constexpr int stage = decltype(stage_)::value;
            const int t = t0 + n % per;
            if (tid < BM) { stat[stage][0][tid] = sl; stat[stage][1][tid] = sd; }
            qg.template arrived<GUARD>(stage);
            __syncthreads();
            if (n + 1 < turns) fetch(n + 1, stage ^ 1);
            if ((t + 1) * BM <= wave_first) return;
            const bool hidden = t * BM < wave_all || (t + 1) * BM > rows.count;   // (zeros stand for rows behind the last: 0 * inf)
            const char *qs = qg.first(stage), *gs = qg.second(stage);
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    const frag_t<T> qf = L::rows(qs, 32 * b + r, st, h), gf = L::rows(gs, 32 * b + r, st, h);
                    s = GUARD ? mma_any<T>(qf, kf[st], s, h) : mma(qf, kf[st], s);
                    dp = GUARD ? mma_any<T>(gf, vf[st], dp, h) : mma(gf, vf[st], dp);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 l4 = *reinterpret_cast<const f32x4*>(&stat[stage][0][32 * b + 8 * g + 4 * h]);
                    const f32x4 d4 = *reinterpret_cast<const f32x4*>(&stat[stage][1][32 * b + 8 * g + 4 * h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * g + e;
                        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, -l4[e]));
                        dp[i] = s[i] * (dp[i] - d4[e]);
                    }
                }
                // element n & 7 of half n >> 3 of step tt stands for token t BM + 32 b + 16 tt + 8 (n >> 2 & 1) + 4 (n >> 3) + (n & 3)
                const int tok0 = t * BM + 32 * b;
                if (hidden) {
                    const int lo = first - tok0 - 4 * h, hi = rows.count - tok0 - 4 * h;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int x = 8 * (i >> 2) + (i & 3);
                        s[i] = seen_or(seen_or(s[i], 0.f, -1 - x, -lo), 0.f, x, hi);
                        dp[i] = seen_or(seen_or(dp[i], 0.f, -1 - x, -lo), 0.f, x, hi);
                    }
                }
                in_range<T, DB>(dp, dk, e);
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const frag_t<T> pf = to_frag<T>(s, tt), df = to_frag<T>(dp, tt);   // rounded to the rows' type for the products with them
                    const int r0 = 32 * b + 16 * tt;
                    const auto sees = [&](int m) {
                        const int tok = tok0 + 16 * tt + 8 * ((m >> 2) & 1) + 4 * (m >> 3) + (m & 3);
                        return tok >= first && tok < rows.count;
                    };
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const frag_t<T> gt = L::cols(gs, r0, 32 * d, lane);
                        if constexpr (!GUARD) dv[d] = mma(gt, pf, dv[d]);
                        else dv[d] = mma_hidden<T>(gt, pf, dv[d], h, sees);
                    }
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const frag_t<T> qt = L::cols(qs, r0, 32 * d, lane);
                        if constexpr (!GUARD) dk[d] = mma(qt, df, dk[d]);
                        else dk[d] = mma_hidden<T>(qt, df, dk[d], h, sees);
                    }
                }
            }
        };
        for (int n = n0; n < turns; n += 2) {
            step(n, std::integral_constant<int, 0>{});
            if (n + 1 < turns) step(n + 1, std::integral_constant<int, 1>{});
        }
    };
    pass(std::false_type{});
    if (a.s.causal || std::is_same<T, x3_t>::value) {
        if (__syncthreads_or(not_finite(dk) || not_finite(dv))) pass(std::true_type{});
    }
    if (key >= share.count) return;
    const long long out_row = (long long)(share.begin + key) * a.Hk + hk;
    if (!used) {
#pragma unroll
        for (int d = 0; d < DB; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
    }
    const float fk = out_of_range<T>(a.scale, e, P_BITS<T>), fv = out_of_range<T>(1.f, 0, P_BITS<T>);
    if (a.splits > 1) {
        const long long n = a.s.Tk * a.Hk * a.D;
        float* part = a.part + 2 * n * blockIdx.y + out_row * a.D;
        store_row<float, DB>(part, dk, h, a.D, fk);
        store_row<float, DB>(part + n, dv, h, a.D, fv);
        return;
    }
    store_row<store_t<T>, DB>((store_t<T>*)a.dk + out_row * a.D, dk, h, a.D, fk);
    store_row<store_t<T>, DB>((store_t<T>*)a.dv + out_row * a.D, dv, h, a.D, fv);
}

// dk and dv as the sums of their splits, in order
template <typename T>
__global__ __launch_bounds__(256) void packed_attn_dkv_join_kernel(const BwdArgs a) {
    const long long n = a.s.Tk * a.Hk * a.D, i = 8 * ((long long)blockIdx.x * 256 + threadIdx.x);
    if (i >= n) return;
    const int m = (int)min(8LL, n - i);
    const float* part = a.part + (blockIdx.y ? n : 0) + i;
    float v[8], x[8];
    load_n(part, v, m);
    for (int s = 1; s < a.splits; ++s) {
        load_n(part + 2 * n * s, x, m);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += x[e];
    }
    store_n((T*)(blockIdx.y ? a.dv : a.dk) + i, v, m);
}

constexpr int BWD_NW = 4;

// Parts that the rows of a key tile are split into.  A key tile walks all rows of all the heads that share it, so few key heads leave the chip to
// a few long workgroups; each part costs a write and a read of dk and dv in fp32.  6 packed documents up to 4096, 4 key heads of 64, 432 key
// tiles, both kernels with parts for at least 512 / 768 / 1024 / 1400 / 2048 workgroups: 346 / 339 / 307 / 327 / 316 us.
int split_rows(long long Tk, int n, int Hk) {
    const long long wgs = slot_count(Tk, 1, n, 32 * BWD_NW) * Hk;
    return wgs >= 1024 ? 1 : (int)(wgs >= 128 ? 1 + 1023 / wgs : 8);
}
}  // namespace

extern "C" size_t casmtr_packed_attn_bwd_ws_floats(long long Tq, long long Tk, int nseq, int H, int Hk, int D) {
    if (Tq <= 0 || Tk < 0 || nseq < 0 || H <= 0 || Hk <= 0 || D <= 0) return 0;
    const int s = split_rows(Tk, nseq, Hk);
    return (size_t)Tq * H + (s > 1 ? (size_t)2 * s * Tk * Hk * D + 3 : 0);
}

extern "C" int casmtr_packed_attn_bwd(const void* g, const void* q, const void* k, const void* v, const void* o, const float* lse, void* dq, void* dk,
                                      void* dv, float* ws, const int* cu_q, const int* cu_k, const int* len_k, long long Tq, long long Tk, int nseq,
                                      int H, int Hk, int D, long long qts, long long qhs, long long kts, long long khs, long long vts, long long vhs,
                                      float scale, int causal, int dtype, casmtr_stream_t stream) {
    if (Tq < 0 || Tk < 0 || nseq < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || D <= 0 || D > 128 || !(scale > 0.f) || !(scale * LOG2E < INFINITY) ||
        Tq > 0x7fffff00LL || Tk > 0x7fffff00LL || Tq * (H / Hk) > 0x7fffff00LL || dtype < 0 || dtype > CASMTR_BF16)
        return CASMTR_ERR_UNSUPPORTED;
    if (Tq == 0 && Tk == 0) return 0;
    const int G = H / Hk;
    const long long qwgs = slot_count(Tq, G, nseq, 32 * BWD_NW) * Hk, kwgs = slot_count(Tk, 1, nseq, 32 * BWD_NW) * Hk;
    if (qwgs > 0x7fffffffLL || kwgs > 0x7fffffffLL) return CASMTR_ERR_UNSUPPORTED;
    if (Tq > 0 && (!ws || !lse)) return CASMTR_ERR_UNSUPPORTED;
    const int splits = Tq > 0 ? split_rows(Tk, nseq, Hk) : 1;
    float* part = ws ? ws + (((size_t)Tq * H + 3) & ~(size_t)3) : nullptr;
    BwdArgs a{q, k, v, o, g, lse, ws, part, dq, dk, dv, {cu_q, cu_k, len_k, nseq, G, causal != 0, Tq, Tk}, qts, qhs, kts, khs, vts, vhs, H, Hk, D, splits,
              scale, scale * LOG2E};
    ProfScope ps(CASMTR_PROF_GLUE, (hipStream_t)stream, "packed_attn_dq_kernel, packed_attn_dkv_kernel");
    with_type(dtype, [&](auto tv) {
        typedef decltype(tv) T;
        const dim3 block(64 * BWD_NW), qgrid((unsigned)qwgs), kgrid((unsigned)kwgs, (unsigned)splits);
        const hipStream_t st = (hipStream_t)stream;
        typedef TileDma<T, 128, 64, BWD_NW> Dma;
        const bool kdma = Dma::fits(k, kts, khs, D) && Dma::fits(v, vts, vhs, D), qdma = Dma::fits(q, qts, qhs, D) && Dma::fits(g, (long long)H * D, D, D);
        // E: the element as the kernel multiplies it (x3_t: fp32 in three terms, staged through registers at any alignment)
#define BWD_LAUNCH(KERNEL, E, DP, TILE, DMA, GRID)                                                                      \
    do {                                                                                                                \
        constexpr bool CAN = sizeof(E) != 1;                                                                            \
        if (CAN && DMA) hipLaunchKernelGGL((KERNEL<E, DP, TILE, BWD_NW, CAN>), GRID, block, 0, st, a);                  \
        else hipLaunchKernelGGL((KERNEL<E, DP, TILE, BWD_NW, false>), GRID, block, 0, st, a);                           \
    } while (0)
        constexpr bool WIDE = sizeof(T) == 4;
        typedef std::conditional_t<WIDE, x3_t, T> E;
        if (Tq > 0) {
            if (D <= 32) BWD_LAUNCH(packed_attn_dq_kernel, E, 32, 64, kdma, qgrid);
            else if (D <= 64) BWD_LAUNCH(packed_attn_dq_kernel, E, 64, (WIDE ? 32 : 64), kdma, qgrid);
            else BWD_LAUNCH(packed_attn_dq_kernel, E, 128, (WIDE ? 32 : 64), kdma, qgrid);
        }
        if (Tk > 0) {
            if (D <= 32) BWD_LAUNCH(packed_attn_dkv_kernel, E, 32, 64, qdma, kgrid);
            else if (D <= 64) BWD_LAUNCH(packed_attn_dkv_kernel, E, 64, (WIDE ? 32 : 64), qdma, kgrid);
            else BWD_LAUNCH(packed_attn_dkv_kernel, T, 128, (WIDE ? 32 : 64), qdma, kgrid);   // fp32 terms of K and V do not fit the registers here: 95 against 124 TFLOP/s
        }
#undef BWD_LAUNCH
        if (splits > 1 && Tk > 0)
            hipLaunchKernelGGL((packed_attn_dkv_join_kernel<T>), dim3((unsigned)((Tk * Hk * D + 2047) / 2048), 2), dim3(256), 0, st, a);
    });
    CASMTR_CHECK_LAUNCH();
    return 0;
}
