// softmax(Q K^T * scale) V over packed sequences of different lengths with grouped heads, the keys and values packed like
// the queries (whole prompts) or in the pages of a cache (chunks of new tokens, single tokens).
//
// Rows.  The query heads that share a key / value head read the same keys, so the rows of a tile are (token, head of the
// group) pairs of one sequence and one key / value head, token-major: row rr of a sequence of n tokens is token rr / G,
// head rr % G, rr < n G.  A tile takes consecutive rows; a key is then fetched once for all heads of the group, a
// single token of a group of 8 fills half a tile instead of a sixteenth, and a causal tile covers few tokens, so
// little of it lies behind the mask.  The number of tiles is known to the host up to the sequences' raggedness
// (rows / tile + one per sequence); which sequence a tile belongs to is found on the device from the offsets.
//
// Row i of n over m keys attends keys 0 .. i + m - n (causal) or all m.  In f32, per row, over the keys in any order:
//   m' = max(m, s)   l' = l 2^(c (m - m')) + 2^(c (s - m'))   o' = o 2^(c (m - m')) + 2^(c (s - m')) v,  c = scale log2 e
// and o / l at the end: one pass, scores never leave the chip.
#include <type_traits>

#include "common.hpp"
#include "device_types.hpp"
#include "gemm_mfma_pipe.hpp"
#include "gfx950_insn.hpp"

namespace hodu {
namespace {

using mfma::Compute;
using mfma::lds_get;
using mfma::lds_get64;
using mfma::lds_get_tr;

struct DevSeq {
    int batch, q_tokens, k_tokens, heads, kv_heads, group;
    int n_pages, width;
    FixedDiv page;   // tokens of a page
    FixedDiv by_group;
    long q_token, q_head;
    PagedSide kc, vc;  // in BYTES
    const int *q_offsets, *k_offsets, *table, *lens;
    const float *k_scale, *v_scale;
    float scale_log2e;
    int causal;
};

__device__ __forceinline__ int quot(int n, const FixedDiv &f) { return (int)(((unsigned long long)(unsigned)n * f.mul) >> f.sh); }

// what lane `from` of the wavefront holds
__device__ __forceinline__ int from_lane(int v, int from) { return __builtin_amdgcn_ds_bpermute(from << 2, v); }

// The sequence and first row of tile `tile` of `rows` rows (found by the whole wavefront, the same in all lanes); false
// past the last tile.  n: the sequence's tokens, q0: its first one
template <int ROWS> __device__ __forceinline__ bool find_tile(const DevSeq &a, int tile, int &b, int &row0, int &q0, int &n) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.batch; base += 64) {
        const int s = base + lane;
        int lo = 0, len = 0;
        if (s < a.batch) {
            lo = a.q_offsets[s];
            const int hi = a.q_offsets[s + 1] < a.q_tokens ? a.q_offsets[s + 1] : a.q_tokens;
            lo = lo > 0 ? lo : 0;
            len = hi > lo ? hi - lo : 0;
        }
        const int tiles = (int)(((long)len * a.group + ROWS - 1) / ROWS);
        int sum = tiles;  // inclusive over the lanes
#pragma unroll
        for (int step = 1; step < 64; step *= 2) {
            const int up = from_lane(sum, lane >= step ? lane - step : lane);
            sum += lane >= step ? up : 0;
        }
        const int all = from_lane(sum, 63);
        if (tile < before + all) {
            const unsigned long long past = __builtin_amdgcn_ballot_w64(before + sum > tile);
            const int at = __builtin_ctzll(past);
            b = base + at;
            const int first = before + from_lane(sum, at) - from_lane(tiles, at);
            q0 = from_lane(lo, at);
            n = from_lane(len, at);
            row0 = (tile - first) * ROWS;
            b = __builtin_amdgcn_readfirstlane(b);
            q0 = __builtin_amdgcn_readfirstlane(q0);
            n = __builtin_amdgcn_readfirstlane(n);
            row0 = __builtin_amdgcn_readfirstlane(row0);
            // (offsets that do not ascend can make the count above wrap; a tile outside its sequence is no tile)
            return row0 >= 0 && row0 < (long)n * a.group;
        }
        before += all;
    }
    return false;
}

// keys of sequence b and, packed, where they begin
template <bool PAGED> __device__ __forceinline__ void find_keys(const DevSeq &a, int b, int &k0, int &m) {
    if constexpr (PAGED) {
        k0 = 0;
        const int most = a.width * a.page.d, len = a.lens[b];
        m = len < 0 ? 0 : len < most ? len : most;
    } else {
        k0 = a.k_offsets[b];
        const int hi = a.k_offsets[b + 1] < a.k_tokens ? a.k_offsets[b + 1] : a.k_tokens;
        k0 = k0 > 0 ? k0 : 0;
        m = hi > k0 ? hi - k0 : 0;
    }
    k0 = __builtin_amdgcn_readfirstlane(k0);
    m = __builtin_amdgcn_readfirstlane(m);
}

template <int CK> __device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    if constexpr (CK == mfma::CK_BF16) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
    }
}

// 8 f8e4m3 -> 8 of the compute type, exact (every e4m3 value is a bf16 and an f16 value)
template <int CK> __device__ __forceinline__ u32x4_t widen8(const u32x2_t &v) {
    if constexpr (CK == mfma::CK_BF16) {
        return mfma::widen_f8x8(v);
    } else {
        return u32x4_t{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.x, 1.0f, false)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.x, 1.0f, true)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.y, 1.0f, false)),
                       __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(v.y, 1.0f, true))};
    }
}

// ---- tiles of 16 rows, one wavefront at a time over a range of the keys -------------------------------------------------
// A workgroup is four wavefronts with the same 16 rows and a quarter of the keys each, 32 keys at a step; they meet once, at the end, in
// LDS.  S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32: a lane then owns one row throughout (column lane % 16).  The rows
// of the first product's left operand are keys in the order 8 (r / 4) + 4 t + r % 4 for tile t of two, so that a lane's
// eight scores are those of 8 consecutive keys -- which is the operand layout of P in the second product, and the order
// in which the LDS transpose reads deliver V's keys.  K and V blocks go from memory into LDS without registers in between,
// rows back to back, 16-byte chunks XOR-swizzled on the source side so that the rows of one read fall into different banks.
constexpr int R16 = 16, R16_NT = 256, R16_BK = 32;
template <int D, bool F8> struct R16Geom {
    static_assert(D == 64 || D == 128, "head dim");
    static constexpr int ES = F8 ? 1 : 2, ROW = D * ES, CPR = ROW / 16, BLOCK = R16_BK * ROW, DMAS = BLOCK / 1024, KPI = 64 / CPR;
    static constexpr int KS = D / 32, DT = D / 16;  // 32-wide slices of the head dim, 16-wide tiles of the output
    // A read's lanes go through keys that differ in bits {0, 1, 3, 4} (K: 16 keys of a tile, one chunk each), {0, 1, 3} (V, 16-bit:
    // 8 keys, two chunks each), {0, 1, 2, 3} (V, 8-bit: 16 keys, a chunk each); the lowest bits choose the row's part of the
    // 64 banks already (256 / ROW rows lie side by side), the others go into the chunk index
    static __device__ __forceinline__ int kswz(int key) {
        const int bits = (key & 3) | ((key >> 1) & 12);
        return ROW == 256 ? bits : ROW == 128 ? bits >> 1 : bits >> 2;
    }
    static __device__ __forceinline__ int vswz(int key) {
        if (F8) return ROW == 128 ? (key >> 1) & 7 : (key >> 2) & 3;
        const int bits = (key & 3) | ((key >> 1) & 4);
        return (ROW == 256 ? bits : bits >> 1) << 1;
    }
    static constexpr int WAVE = 2 * BLOCK;                   // a wavefront's K and V block
    static constexpr int MERGE = 4 * R16 * (D + 4) * 4;      // (m, l, O) of four wavefronts
    static constexpr int LDS = 4 * WAVE > MERGE ? 4 * WAVE : MERGE;
};

template <int CK, int D, bool PAGED, bool F8>
__global__ __launch_bounds__(R16_NT) void seq_attention_r16_kernel(const uint16_t *__restrict__ Q, const char *__restrict__ K,
                                                                   const char *__restrict__ V, uint16_t *__restrict__ O, DevSeq a) {
    typedef R16Geom<D, F8> G;
    typedef Compute<CK> Cmp;
    typedef typename Cmp::acc_t acc_t;
    HODU_DYNAMIC_LDS(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.kv_heads;
    int b, row0, q0, n, k0, m;
    if (!find_tile<R16>(a, blockIdx.x / a.kv_heads, b, row0, q0, n)) return;
    find_keys<PAGED>(a, b, k0, m);

    // the lane's row; rows past the sequence's last repeat it and are not stored
    const int rows = n * a.group;
    const int rr = row0 + r < rows ? row0 + r : rows - 1;
    const int tok = quot(rr, a.by_group), head = kvh * a.group + rr - tok * a.group;
    const int open = a.causal ? tok + m - n + 1 : m;  // keys the row attends, <= 0: none
    const int last_tok = quot(row0 + R16 - 1 < rows ? row0 + R16 - 1 : rows - 1, a.by_group), first_tok = quot(row0, a.by_group);
    const int keys = a.causal ? last_tok + m - n + 1 : m;          // keys the tile needs
    const int all_open = a.causal ? first_tok + m - n + 1 : m;     // keys below this are open to every row
    const int blocks = keys > 0 ? (keys + R16_BK - 1) / R16_BK : 0;
    const int blk0 = (int)((long)blocks * wave / 4), blk1 = (int)((long)blocks * (wave + 1) / 4);

    u32x4_t qf[G::KS];
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++)
        qf[ks] = *reinterpret_cast<const u32x4_t *>(Q + (q0 + tok) * a.q_token + head * a.q_head + 32 * ks + 8 * g);
    const float c = a.scale_log2e * (F8 ? a.k_scale[kvh] : 1.f);

    char *kl = smem + wave * G::WAVE, *vl = kl + G::BLOCK;
    const unsigned kl0 = (unsigned)(uintptr_t)kl, vl0 = (unsigned)(uintptr_t)vl;
    const char *kbase = K + kvh * a.kc.head, *vbase = V + kvh * a.vc.head;
    int k_frag[2];
#pragma unroll
    for (int t = 0; t < 2; t++) k_frag[t] = 8 * (r >> 2) + 4 * t + (r & 3);
    acc_t o[G::DT];
#pragma unroll
    for (int j = 0; j < G::DT; j++) o[j] = acc_t{0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;

    for (int blk = blk0; blk < blk1; blk++) {
        // the last block's reads have been answered before this one's loads are issued
        __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(63));
        mfma::wave_lds_fence();
#pragma unroll
        for (int i = 0; i < G::DMAS; i++) {
            const int kk = i * G::KPI + lane / G::CPR;  // the lane's key of this instruction
            int key = blk * R16_BK + kk;
            key = key < keys ? key : keys - 1;  // behind the last key: that one again, masked below
            long ko, vo;
            if constexpr (PAGED) {
                const int col = quot(key, a.page), in = key - col * a.page.d;
                int pg = a.table[(long)b * a.width + col];
                pg = pg < 0 ? 0 : pg < a.n_pages ? pg : a.n_pages - 1;
                ko = pg * a.kc.page + in * a.kc.token;
                vo = pg * a.vc.page + in * a.vc.token;
            } else {
                ko = (k0 + key) * a.kc.token;
                vo = (k0 + key) * a.vc.token;
            }
            const int slot = lane % G::CPR;
            mfma::dma16_raw(kbase + ko + ((slot ^ G::kswz(kk)) << 4), __builtin_amdgcn_readfirstlane(kl0 + i * 1024));
            mfma::dma16_raw(vbase + vo + ((slot ^ G::vswz(kk)) << 4), __builtin_amdgcn_readfirstlane(vl0 + i * 1024));
        }
        __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(0));
        mfma::wave_lds_fence();

        acc_t s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = acc_t{0.f, 0.f, 0.f, 0.f};
            const int key = k_frag[t];
#pragma unroll
            for (int ks = 0; ks < G::KS; ks++) {
                u32x4_t kf;
                if constexpr (F8)
                    kf = widen8<CK>(lds_get64(kl, key * G::ROW + (((2 * ks + (g >> 1)) ^ G::kswz(key)) << 4) + (g & 1) * 8));
                else
                    kf = lds_get(kl, key * G::ROW + (((4 * ks + g) ^ G::kswz(key)) << 4));
                Cmp::mma(kf, qf[ks], s[t]);
            }
        }
        // the lane's keys: blk * 32 + 8 g + 0 .. 7
        float sv[8];
#pragma unroll
        for (int e = 0; e < 4; e++) { sv[e] = s[0][e]; sv[4 + e] = s[1][e]; }
        if ((blk + 1) * R16_BK > all_open) {
#pragma unroll
            for (int e = 0; e < 8; e++) sv[e] = blk * R16_BK + 8 * g + e < open ? sv[e] : -INFINITY;
        }
        float mx = sv[0];
#pragma unroll
        for (int e = 1; e < 8; e++) mx = __builtin_fmaxf(mx, sv[e]);
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
        const float m_new = __builtin_fmaxf(m_run, mx);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;  // no key yet: 2^(-inf) = 0 keeps the sums at zero
        const float keep = __builtin_amdgcn_exp2f((m_run - m_use) * c);
        m_run = m_new;
        float p[8], sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            p[e] = __builtin_amdgcn_exp2f((sv[e] - m_use) * c);
            sum += p[e];
        }
        l_run = l_run * keep + sum;  // the lane's share; the row's four lanes add up at the end
        const u32x4_t pf = {pack2<CK>(p[0], p[1]), pack2<CK>(p[2], p[3]), pack2<CK>(p[4], p[5]), pack2<CK>(p[6], p[7])};
#pragma unroll
        for (int j = 0; j < G::DT; j++) {
            u32x4_t vf;
            if constexpr (F8) {
                const int key = 8 * g + (r >> 1);
                vf = widen8<CK>(lds_get_tr<1>(vl, key * G::ROW + ((j ^ G::vswz(key)) << 4) + (r & 1) * 8));
            } else {
                const int key = 8 * g + (r >> 2), ch = 2 * j + ((r >> 1) & 1);
                const u32x2_t lo = lds_get_tr<2>(vl, key * G::ROW + ((ch ^ G::vswz(key)) << 4) + (r & 1) * 8);
                const u32x2_t hi = lds_get_tr<2>(vl, (key + 4) * G::ROW + ((ch ^ G::vswz(key + 4)) << 4) + (r & 1) * 8);
                vf = u32x4_t{lo.x, lo.y, hi.x, hi.y};
            }
#pragma unroll
            for (int e = 0; e < 4; e++) o[j][e] *= keep;
            Cmp::mma(vf, pf, o[j]);
        }
    }

    // ---- the four wavefronts meet: per wavefront and row (m, l, -, -, O) ----
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    __syncthreads();
    constexpr int LINE = D + 4;
    float *mg = reinterpret_cast<float *>(smem);
    {
        float *mine = mg + (wave * R16 + r) * LINE;
        if (g == 0) {
            mine[0] = m_run;
            mine[1] = l_run;
        }
#pragma unroll
        for (int j = 0; j < G::DT; j++) *reinterpret_cast<f32x4_t *>(mine + 4 + 16 * j + 4 * g) = f32x4_t{o[j][0], o[j][1], o[j][2], o[j][3]};
    }
    __syncthreads();
    const int row = tid >> 4, part = tid & 15;  // 16 threads a row, D / 16 elements each
    if (row0 + row >= rows) return;
    float mx = -INFINITY, l = 0.f, w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) mx = __builtin_fmaxf(mx, mg[(i * R16 + row) * LINE]);
    const float c2 = c;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float *line = mg + (i * R16 + row) * LINE;
        w[i] = line[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((line[0] - mx) * c2);
        l += line[1] * w[i];
    }
    // a row without keys: l = 0, and zero is what it gives
    const float inv = l == 0.f ? 0.f : (F8 ? a.v_scale[kvh] : 1.f) / l;
    const int wtok = quot(row0 + row, a.by_group), whead = kvh * a.group + row0 + row - wtok * a.group;
    constexpr int PER = D / 16;
    uint32_t out[PER / 2];
#pragma unroll
    for (int e = 0; e < PER; e += 2) {
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float *line = mg + (i * R16 + row) * LINE + 4 + part * PER + e;
            x += line[0] * w[i];
            y += line[1] * w[i];
        }
        out[e / 2] = pack2<CK>(x * inv, y * inv);
    }
    uint16_t *dst = O + ((long)(q0 + wtok) * a.heads + whead) * D + part * PER;
    if constexpr (PER == 8) *reinterpret_cast<u32x4_t *>(dst) = u32x4_t{out[0], out[1], out[2], out[3]};
    else *reinterpret_cast<u32x2_t *>(dst) = u32x2_t{out[0], out[1]};
}

}  // namespace

int launch_seq_attention(hodu_rocm_ctx *ctx, int dtype, int cache_dtype, const void *q, const void *k, const void *v, void *out,
                         const SeqAttentionArgs &g) {
    if (dtype != HODU_BF16 && dtype != HODU_F16) return HODU_ROCM_UNSUPPORTED;
    if (g.d != 64 && g.d != 128) return HODU_ROCM_UNSUPPORTED;
    // the row maximum is taken before the scale is applied: the scale must be positive (and finite)
    if (!(g.scale > 0.f) || !(g.scale < INFINITY)) return HODU_ROCM_UNSUPPORTED;
    const bool f8 = cache_dtype == HODU_F8E4M3;
    const long es = f8 ? 1 : 2;
    // 16-byte accesses: rows, heads, pages, offsets and bases
    for (long e : {g.q_token, g.q_head, g.q_off})
        if (e % 8) return HODU_ROCM_UNSUPPORTED;
    for (long e : {g.kc.page, g.kc.token, g.kc.head, g.kc.off, g.vc.page, g.vc.token, g.vc.head, g.vc.off})
        if (e * es % 16) return HODU_ROCM_UNSUPPORTED;
    if ((uintptr_t)q % 16 || (uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)out % 16) return HODU_ROCM_UNSUPPORTED;
    DevSeq a{};
    a.batch = (int)g.batch; a.q_tokens = (int)g.q_tokens; a.k_tokens = (int)g.k_tokens;
    a.heads = (int)g.heads; a.kv_heads = (int)g.kv_heads; a.group = (int)(g.heads / g.kv_heads);
    // (a cache without a page holds no key: no table entry is read)
    a.n_pages = (int)g.n_pages; a.width = g.n_pages ? (int)g.width : 0;
    a.page = fixed_div((int)g.page_size);
    a.by_group = fixed_div(a.group);
    a.q_token = g.q_token; a.q_head = g.q_head;
    a.kc = PagedSide{g.kc.page * es, g.kc.token * es, g.kc.head * es, 0};
    a.vc = PagedSide{g.vc.page * es, g.vc.token * es, g.vc.head * es, 0};
    a.q_offsets = g.q_offsets; a.k_offsets = g.k_offsets; a.table = g.table; a.lens = g.lens;
    a.k_scale = g.k_scale; a.v_scale = g.v_scale;
    a.scale_log2e = g.scale * 1.44269504088896340736f;
    a.causal = g.causal ? 1 : 0;
    const uint16_t *qp = (const uint16_t *)q + g.q_off;
    const char *kp = (const char *)k + g.kc.off * es, *vp = (const char *)v + g.vc.off * es;
    const long tiles = (g.q_tokens < g.batch ? g.q_tokens : g.batch) + g.q_tokens * a.group / R16;
    const long blocks = tiles * g.kv_heads;
    if (blocks > 0x7FFFFFFFL) return HODU_ROCM_UNSUPPORTED;
    auto launch = [&](auto kernel, int lds, const char *name) -> int {
        if (int rc = ensure_dynamic_lds(ctx, reinterpret_cast<const void *>(kernel), lds)) return rc;
        ctx->last_kernel = name;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(R16_NT), lds, ctx->stream, qp, kp, vp, (uint16_t *)out, a);
        return HODU_ROCM_OK;
    };
    auto by_type = [&](auto ck, auto d) -> int {
        constexpr int CK = decltype(ck)::value, D = decltype(d)::value;
        if (!g.paged) return launch(seq_attention_r16_kernel<CK, D, false, false>, R16Geom<D, false>::LDS, "attention_varlen_r16");
        if (f8) return launch(seq_attention_r16_kernel<CK, D, true, true>, R16Geom<D, true>::LDS, "attention_paged_r16_f8");
        return launch(seq_attention_r16_kernel<CK, D, true, false>, R16Geom<D, false>::LDS, "attention_paged_r16");
    };
    typedef std::integral_constant<int, 64> d64;
    typedef std::integral_constant<int, 128> d128;
    typedef std::integral_constant<int, mfma::CK_BF16> bf16;
    typedef std::integral_constant<int, mfma::CK_F16> f16;
    int rc;
    if (dtype == HODU_BF16) rc = g.d == 128 ? by_type(bf16(), d128()) : by_type(bf16(), d64());
    else rc = g.d == 128 ? by_type(f16(), d128()) : by_type(f16(), d64());
    if (rc != HODU_ROCM_OK) return rc;
    HODU_HIP(hipGetLastError());
    return HODU_ROCM_OK;
}

}  // namespace hodu
