// Attention over packed sequences, backward.  With p_ij = exp(scale q_i . k_j - lse_i):
//   delta_i = sum_d do_i o_i;  ds_ij = p_ij (do_i . v_j - delta_i) scale
//   dq_i = sum_j ds_ij k_j;    dk_j = sum_i ds_ij q_i;    dv_j = sum_i p_ij do_i
// Two kernels, no atomics: one owns query rows and walks the keys (dq, and delta on the way), one owns keys and walks the query rows of all
// heads that share them (dk, dv: the sum over the group is in the accumulator).  The scores are computed twice for it -- 7 products
// instead of 5 -- and results repeat bit for bit.
#include "packed_attn.hpp"

using namespace casmtr;

namespace {
struct BwdArgs {
    const void *q, *k, *v, *o, *g;     // o, g (the gradient of o): [Tq, H, D] contiguous
    const float* lse;
    float* delta;                      // [Tq, H]
    void *dq, *dk, *dv;                // contiguous
    PackedSeqs s;
    long long qts, qhs, kts, khs, vts, vhs;
    int H, Hk, D;
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

// dq: a workgroup's rows are (token, head) pairs as in the forward kernel
template <typename T, int DP, int BN, int NW>
__global__ __launch_bounds__(64 * NW) void packed_attn_dq_kernel(const BwdArgs a) {
    typedef Tile<T, DP> L;
    constexpr int BM = 32 * NW, NT = 64 * NW, KS = DP / 16, NB = BN / 32, DB = DP / 32;
    constexpr int NCH = BN * L::CPR / NT, TB = BN * L::RB;
    __shared__ __attribute__((aligned(256))) char smem[4 * TB];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, r = lane & 31;
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
    float delta = 0.f;
    {
        const T* qr = (const T*)a.q + (long long)(rows.begin + tok) * a.qts + head * a.qhs;
        const T *gr = (const T*)a.g + out_row * a.D, *orow = (const T*)a.o + out_row * a.D;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = load_frag(qr, s, h, a.D);
            gf[s] = load_frag(gr, s, h, a.D);
            const frag_t<T> of = load_frag(orow, s, h, a.D);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf((float)gf[s][e], (float)of[e], delta);
        }
    }
    delta = add_halves(delta);
    const float lse = a.lse[out_row], lse2 = lse == -INFINITY ? 0.f : lse * LOG2E;   // (a row that sees nothing: every key is hidden below)
    if (h == 0 && row < nrow) a.delta[out_row] = delta;
    f32x16 acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) acc[d] = zero16();

    const T* kb = (const T*)a.k + (long long)keys.begin * a.kts + hk * a.khs;
    const T* vb = (const T*)a.v + (long long)keys.begin * a.vts + hk * a.vhs;
    u32x4 kr[NCH], vr[NCH];
    const auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int id = tid + NT * i, rr = t * BN + id / L::CPR, c = (id % L::CPR) * L::EPC;
            kr[i] = u32x4{0, 0, 0, 0};
            vr[i] = u32x4{0, 0, 0, 0};
            if (rr < keys.count && c < a.D) {
                kr[i] = load_chunk(kb + (long long)rr * a.kts, c, a.D);
                vr[i] = load_chunk(vb + (long long)rr * a.vts, c, a.D);
            }
        }
    };
    const auto put = [&](int stage) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int id = tid + NT * i, o = L::off(id / L::CPR, id % L::CPR);
            *reinterpret_cast<u32x4*>(smem + 2 * stage * TB + o) = kr[i];
            *reinterpret_cast<u32x4*>(smem + (2 * stage + 1) * TB + o) = vr[i];
        }
    };
    if (0 < t1) { fetch(0); put(0); }
    __syncthreads();
    for (int t = 0; t < t1; ++t) {
        const int stage = t & 1;
        if (t + 1 < t1) fetch(t + 1);
        const char *ks = smem + 2 * stage * TB, *vs = ks + TB;
        if (t * BN < wave_end) {
            const bool hidden = (t + 1) * BN > wave_all;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    s = mma(L::rows(ks, 32 * b + r, st, h), qf[st], s);
                    dp = mma(L::rows(vs, 32 * b + r, st, h), gf[st], dp);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, -lse2));
                    s[i] = p * (dp[i] - delta);
                    if (hidden && t * BN + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3) >= limit) s[i] = 0.f;
                }
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const frag_t<T> ds = to_frag<T>(s, tt);   // rounded to the keys' type for the product with them
                    const int k0 = 32 * b + 16 * tt;
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const frag_t<T> kt = L::cols(ks, k0, 32 * d, lane);
                        if (!hidden) acc[d] = mma(kt, ds, acc[d]);
                        else acc[d] = mma_hidden<T>(kt, ds, acc[d], h, [&](int n) { return t * BN + k0 + 8 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3) < limit; });
                    }
                }
            }
        }
        if (t + 1 < t1) put(stage ^ 1);
        __syncthreads();
    }
    if (row < nrow) store_row<T, DB>((T*)a.dq + out_row * a.D, acc, h, a.D, a.scale);
}

// dk, dv: a workgroup owns BN = 32 NW keys of one key head, a wave 32 of them (K and V stay in its registers), and walks the (token, head)
// rows of the group in tiles of BM
template <typename T, int DP, int BM, int NW>
__global__ __launch_bounds__(64 * NW) void packed_attn_dkv_kernel(const BwdArgs a) {
    typedef Tile<T, DP> L;
    constexpr int BN = 32 * NW, NT = 64 * NW, KS = DP / 16, MB = BM / 32, DB = DP / 32;
    constexpr int NCH = BM * L::CPR / NT, TB = BM * L::RB;
    static_assert(BM <= NT, "a thread stages one row's statistics");
    __shared__ __attribute__((aligned(256))) char smem[4 * TB];          // q, g of two stages
    __shared__ __attribute__((aligned(16))) float stat[2][2][BM];        // lse (in bits), delta of two stages
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = lane >> 5, r = lane & 31;
    const int hk = blockIdx.x % a.Hk, G = a.s.G;
    int tile;
    const int seq = seq_of_slot(a.s.cu_k, a.s.n, a.s.Tk, 1, BN, (long long)(blockIdx.x / a.Hk), &tile);   // earlier keys are seen by more rows: first
    const Span share = span_of(a.s.cu_k, seq, a.s.n, a.s.Tk), keys = keys_of(a.s, seq);
    const Span rows = seq >= 0 && seq < a.s.n ? span_of(a.s.cu_q, seq, a.s.n, a.s.Tq) : Span{0, 0};
    if ((long long)tile * BN >= share.count) return;
    const int key0 = tile * BN, key = key0 + 32 * wave + r;      // keys of the share that are not in use get zero gradients
    const int shift = keys.count - rows.count, nrow = rows.count * G;
    const bool used = key < keys.count;
    const int first = !used ? 0x7fffffff : a.s.causal ? max(0, key - shift) : 0;   // this lane's key is seen by the tokens [first, count)
    // tokens that see some key of the workgroup / the wave, tokens that see all of the wave's keys
    const int wg_first = key0 >= keys.count ? rows.count : a.s.causal ? min(rows.count, max(0, key0 - shift)) : 0;
    const int wk = key0 + 32 * wave;
    const int wave_first = wk >= keys.count ? rows.count : a.s.causal ? min(rows.count, max(0, wk - shift)) : 0;
    const int wave_all = wk + 32 > keys.count ? 0x7fffffff : a.s.causal ? max(0, wk + 31 - shift) : 0;
    const int kc = max(0, min(key, keys.count - 1));
    frag_t<T> kf[KS], vf[KS];
    {
        const T* kr = (const T*)a.k + (long long)(keys.begin + kc) * a.kts + hk * a.khs;
        const T* vr = (const T*)a.v + (long long)(keys.begin + kc) * a.vts + hk * a.vhs;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            kf[s] = load_frag(kr, s, h, keys.count > 0 ? a.D : 0);
            vf[s] = load_frag(vr, s, h, keys.count > 0 ? a.D : 0);
        }
    }
    f32x16 dk[DB], dv[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) { dk[d] = zero16(); dv[d] = zero16(); }

    const int t0 = (int)((long long)wg_first * G / BM), t1 = (nrow + BM - 1) / BM;
    u32x4 qr[NCH], gr[NCH];
    float sl = 0.f, sd = 0.f;
    const auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int id = tid + NT * i, rr = t * BM + id / L::CPR, c = (id % L::CPR) * L::EPC;
            qr[i] = u32x4{0, 0, 0, 0};
            gr[i] = u32x4{0, 0, 0, 0};
            if (rr < nrow && c < a.D) {
                const int tok = rr / G, head = hk * G + rr % G;
                qr[i] = load_chunk((const T*)a.q + (long long)(rows.begin + tok) * a.qts + head * a.qhs, c, a.D);
                gr[i] = load_chunk((const T*)a.g + ((long long)(rows.begin + tok) * a.H + head) * a.D, c, a.D);
            }
        }
        if (tid < BM) {
            const int rr = t * BM + tid;
            sl = sd = 0.f;
            if (rr < nrow) {
                const long long at = (long long)(rows.begin + rr / G) * a.H + hk * G + rr % G;
                const float x = a.lse[at];
                sl = x == -INFINITY ? 0.f : x * LOG2E;
                sd = a.delta[at];
            }
        }
    };
    const auto put = [&](int stage) {
#pragma unroll
        for (int i = 0; i < NCH; ++i) {
            const int id = tid + NT * i, o = L::off(id / L::CPR, id % L::CPR);
            *reinterpret_cast<u32x4*>(smem + 2 * stage * TB + o) = qr[i];
            *reinterpret_cast<u32x4*>(smem + (2 * stage + 1) * TB + o) = gr[i];
        }
        if (tid < BM) { stat[stage][0][tid] = sl; stat[stage][1][tid] = sd; }
    };
    if (t0 < t1) { fetch(t0); put(0); }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int stage = (t - t0) & 1;
        if (t + 1 < t1) fetch(t + 1);
        const char *qs = smem + 2 * stage * TB, *gs = qs + TB;
        if (min((t + 1) * BM - 1, nrow - 1) / G >= wave_first && wave_first < rows.count) {
            const bool hidden = t * BM / G < wave_all || (t + 1) * BM > nrow;
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int st = 0; st < KS; ++st) {
                    s = mma(L::rows(qs, 32 * b + r, st, h), kf[st], s);
                    dp = mma(L::rows(gs, 32 * b + r, st, h), vf[st], dp);
                }
                unsigned vis = 0xffffu;   // registers whose row sees this lane's key
                if (hidden) {
                    vis = 0;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int rr = t * BM + 32 * b + 8 * (i >> 2) + 4 * h + (i & 3);
                        vis |= (rr < nrow && rr / G >= first ? 1u : 0u) << i;
                    }
                }
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 l4 = *reinterpret_cast<const f32x4*>(&stat[stage][0][32 * b + 8 * g + 4 * h]);
                    const f32x4 d4 = *reinterpret_cast<const f32x4*>(&stat[stage][1][32 * b + 8 * g + 4 * h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * g + e;
                        const bool on = (vis >> i) & 1u;
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], a.scale_log2, -l4[e]));
                        s[i] = on ? p : 0.f;
                        dp[i] = on ? p * (dp[i] - d4[e]) : 0.f;
                    }
                }
#pragma unroll
                for (int tt = 0; tt < 2; ++tt) {
                    const frag_t<T> pf = to_frag<T>(s, tt), df = to_frag<T>(dp, tt);   // rounded to the rows' type for the products with them
                    const int r0 = 32 * b + 16 * tt;
                    // element n & 7 of half n >> 3 stands for row r0 + 8 (n >> 2 & 1) + 4 (n >> 3) + (n & 3)
                    const auto sees = [&](int n) {
                        const int rr = t * BM + r0 + 8 * ((n >> 2) & 1) + 4 * (n >> 3) + (n & 3);
                        return rr < nrow && rr / G >= first;
                    };
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        const frag_t<T> gt = L::cols(gs, r0, 32 * d, lane), qt = L::cols(qs, r0, 32 * d, lane);
                        if (!hidden) {
                            dv[d] = mma(gt, pf, dv[d]);
                            dk[d] = mma(qt, df, dk[d]);
                        } else {
                            dv[d] = mma_hidden<T>(gt, pf, dv[d], h, sees);
                            dk[d] = mma_hidden<T>(qt, df, dk[d], h, sees);
                        }
                    }
                }
            }
        }
        if (t + 1 < t1) put(stage ^ 1);
        __syncthreads();
    }
    if (key >= share.count) return;
    const long long out_row = (long long)(share.begin + key) * a.Hk + hk;
    if (!used) {
#pragma unroll
        for (int d = 0; d < DB; ++d) { dk[d] = zero16(); dv[d] = zero16(); }
    }
    store_row<T, DB>((T*)a.dk + out_row * a.D, dk, h, a.D, a.scale);
    store_row<T, DB>((T*)a.dv + out_row * a.D, dv, h, a.D, 1.f);
}

constexpr int BWD_NW = 4;
}  // namespace

extern "C" int casmtr_packed_attn_bwd(const void* g, const void* q, const void* k, const void* v, const void* o, const float* lse, void* dq, void* dk,
                                      void* dv, float* delta, const int* cu_q, const int* cu_k, const int* len_k, long long Tq, long long Tk, int nseq,
                                      int H, int Hk, int D, long long qts, long long qhs, long long kts, long long khs, long long vts, long long vhs,
                                      float scale, int causal, int dtype, casmtr_stream_t stream) {
    if (Tq < 0 || Tk < 0 || nseq < 0 || H <= 0 || Hk <= 0 || H % Hk != 0 || D <= 0 || D > 128 || !(scale > 0.f) || !(scale < INFINITY) ||
        Tq * (H / Hk) > 0x7fffffffLL || Tk > 0x7fffffffLL || Tq > 0x7fffffffLL || dtype < 0 || dtype > CASMTR_BF16)
        return CASMTR_ERR_UNSUPPORTED;
    if (Tq == 0 && Tk == 0) return 0;
    const int G = H / Hk;
    const long long qwgs = slot_count(Tq, G, nseq, 32 * BWD_NW) * Hk, kwgs = slot_count(Tk, 1, nseq, 32 * BWD_NW) * Hk;
    if (qwgs > 0x7fffffffLL || kwgs > 0x7fffffffLL) return CASMTR_ERR_UNSUPPORTED;
    BwdArgs a{q, k, v, o, g, lse, delta, dq, dk, dv, {cu_q, cu_k, len_k, nseq, G, causal != 0, Tq, Tk}, qts, qhs, kts, khs, vts, vhs, H, Hk, D, scale,
              scale * LOG2E};
    ProfScope ps(CASMTR_PROF_GLUE, (hipStream_t)stream, "packed_attn_dq_kernel, packed_attn_dkv_kernel");
    with_type(dtype, [&](auto tv) {
        typedef decltype(tv) T;
        const dim3 block(64 * BWD_NW);
        constexpr int W = sizeof(T) == 2 ? 64 : 32;   // the widest head's tiles: 64 KB of LDS either way
#define BWD_LAUNCH(DP, TILE, RTILE)                                                                                                                     \
    do {                                                                                                                                         \
        if (Tq > 0) hipLaunchKernelGGL((packed_attn_dq_kernel<T, DP, TILE, BWD_NW>), dim3((unsigned)qwgs), block, 0, (hipStream_t)stream, a);    \
        if (Tk > 0) hipLaunchKernelGGL((packed_attn_dkv_kernel<T, DP, RTILE, BWD_NW>), dim3((unsigned)kwgs), block, 0, (hipStream_t)stream, a);     \
    } while (0)
        if (D <= 32) BWD_LAUNCH(32, 64, 64);
        else if (D <= 64) BWD_LAUNCH(64, 64, 32);
        else BWD_LAUNCH(128, W, 32);
#undef BWD_LAUNCH
    });
    CASMTR_CHECK_LAUNCH();
    return 0;
}
