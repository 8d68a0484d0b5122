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

#include "agent_scope.hpp"
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

__device__ __forceinline__ int quot(int n, const FixedDiv &f) { return fixed_quotient(n, f); }
// keys 0 .. this that token `tok` of n attends of m, causal; <= 0: none.  (In this order no step leaves 31 bits.)
__device__ __forceinline__ int attended(int tok, int n, int m) { return m - (n - 1 - tok); }

// inclusive running sum over the wavefront's lanes (each step one instruction: shifts by 1, 2, 4, 8 within rows of 16 lanes, then
// each row's last lane to the next row, then lane 31 to the upper half)
__device__ __forceinline__ int running_sum64(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// The sequence and first row of tile `tile` of `rows` rows (found by the whole wavefront, the same in all lanes); false
// past the last tile.  n: the sequence's tokens, q0: its first one; m: its keys and, packed, k0: where they begin.
// Every workgroup searches for itself, four sequences a lane, 256 at a step (a step is a trip to memory; a serving batch is one or two).
struct SeqTile {
    int b, row0, q0, n, k0, m;
};
template <int ROWS, bool PAGED> __device__ __forceinline__ bool find_tile(const DevSeq &a, int tile, SeqTile &f) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < a.batch; base += 256) {
        const int s0 = base + 4 * lane;
        int q[5], k[5], tiles[4], lo[4], len[4], own = 0;
#pragma unroll
        for (int i = 0; i < 5; i++) {
            const int s = s0 + i < a.batch ? s0 + i : a.batch;  // (there are batch + 1 offsets)
            q[i] = a.q_offsets[s];
            if constexpr (PAGED) k[i] = a.lens[s < a.batch ? s : a.batch - 1];
            else k[i] = a.k_offsets[s];
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int hi = q[i + 1] < a.q_tokens ? q[i + 1] : a.q_tokens;
            lo[i] = q[i] > 0 ? q[i] : 0;
            len[i] = s0 + i < a.batch && hi > lo[i] ? hi - lo[i] : 0;
            tiles[i] = (int)(((long)len[i] * a.group + ROWS - 1) / ROWS);
            own += tiles[i];
        }
        const int sum = running_sum64(own), all = __builtin_amdgcn_readlane(sum, 63);
        if (tile < before + all) {
            const unsigned long long past = __builtin_amdgcn_ballot_w64(before + sum > tile);
            const int at = __builtin_ctzll(past);
            int left = tile - (before + __builtin_amdgcn_readlane(sum - own, at)), i = 0, t[4];
#pragma unroll
            for (int j = 0; j < 4; j++) t[j] = __builtin_amdgcn_readlane(tiles[j], at);
#pragma unroll
            for (int j = 0; j < 3; j++)
                if (i == j && left >= t[j]) left -= t[j], i = j + 1;
            f.b = base + 4 * at + i;
            f.row0 = left * ROWS;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i == j) {
                    f.q0 = __builtin_amdgcn_readlane(lo[j], at);
                    f.n = __builtin_amdgcn_readlane(len[j], at);
                    const int ka = PAGED ? 0 : __builtin_amdgcn_readlane(k[j], at), kb = __builtin_amdgcn_readlane(k[PAGED ? j : j + 1], at);
                    const int most = PAGED ? a.width * a.page.d : a.k_tokens, k_hi = kb < most ? kb : most;
                    f.k0 = ka > 0 ? ka : 0;
                    f.m = k_hi > f.k0 ? k_hi - f.k0 : 0;
                }
            // (offsets that do not ascend can make the count above wrap; a tile outside its sequence is no tile)
            return f.row0 >= 0 && f.row0 < (long)f.n * a.group;
        }
        before += all;
    }
    return false;
}

// The same for tiles that work for long, of up to 64 sequences: the ones with most keys first and each from its last row, so that
// the tiles left over at a launch's end are short ones (in the sequences' own order and with it: 8192 tokens 679 and 594 us, four chunks of
// 512 over up to 8192 390 and 361, 64 single tokens over up to 8192 270 and 254, 16 packed prompts 421 and 413).  Above 64, one sequence a
// lane does not do, and the sequences' own order is taken: the same requests with an empty one more than 64 cost, this order and that, 255
// and 286 us (64 single tokens over up to 8192), 81 and 88 (over up to 2048), 175 and 185 (64 chunks of 64), but 661 and 612 (64 prompts of up
// to 1024).  A lane owns a sequence, sums the tiles of those before it in that order, and
// knows whether the tile is its own.
template <int ROWS, bool PAGED> __device__ __forceinline__ bool find_tile_long_first(const DevSeq &a, int tile, SeqTile &f) {
    const int lane = threadIdx.x & 63, s = lane < a.batch ? lane : a.batch - 1;
    const int q = a.q_offsets[s], q_end = a.q_offsets[s + 1];
    const int k = PAGED ? 0 : a.k_offsets[s], k_end = PAGED ? a.lens[s] : a.k_offsets[s + 1];
    const int hi = q_end < a.q_tokens ? q_end : a.q_tokens, lo = q > 0 ? q : 0;
    const int len = lane < a.batch && hi > lo ? hi - lo : 0;
    const int most = PAGED ? a.width * a.page.d : a.k_tokens, k_hi = k_end < most ? k_end : most, k0 = k > 0 ? k : 0;
    const int m = k_hi > k0 ? k_hi - k0 : 0;
    const int tiles = (int)(((long)len * a.group + ROWS - 1) / ROWS);
    const unsigned order = ((unsigned)(m < (1 << 26) ? m : (1 << 26) - 1) << 6) + (63 - lane);
    int start = 0;
    for (int j = 0; j < a.batch; j++) {
        const unsigned other = (unsigned)__builtin_amdgcn_readlane((int)order, j);
        const int its = __builtin_amdgcn_readlane(tiles, j);
        start += other > order ? its : 0;
    }
    const unsigned long long mine = __builtin_amdgcn_ballot_w64(tile >= start && tile - start < tiles);
    if (!mine) return false;
    const int at = __builtin_ctzll(mine);
    f.b = at;
    f.row0 = (__builtin_amdgcn_readlane(tiles, at) - 1 - (tile - __builtin_amdgcn_readlane(start, at))) * ROWS;
    f.q0 = __builtin_amdgcn_readlane(lo, at);
    f.n = __builtin_amdgcn_readlane(len, at);
    f.k0 = __builtin_amdgcn_readlane(k0, at);
    f.m = __builtin_amdgcn_readlane(m, at);
    // (offsets that do not ascend can make the sums above wrap; a tile outside its sequence is no tile)
    return f.row0 >= 0 && f.row0 < (long)f.n * a.group;
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

// ---- tiles of 16 rows: single tokens and short chunks ---------------------------------------------------------------------
// Bound by the cache's bytes, or, where there are few of them, by latency.  A workgroup is four wavefronts with the same 16
// rows; the keys of a tile are cut into ranges of 32-key blocks, one per wavefront of each of the tile's workgroups, so that a single long
// sequence still reaches every compute unit.  A wavefront has an LDS ring of its own (32 KB: the next block or blocks are in flight while it computes,
// 64 KB and more per compute unit), meets nobody until its range is done, and there is no barrier in the loop.
// Measured, bf16, 32 query and 8 key / value heads of 128: 64 tokens over up to 8192 cached each, 1.44 GB, 253 us (5.7 TB/s; a
// large copy 5.1, reading alone 7.0); 48 over up to 16384 in 8-bit floats, 64 query heads, 1.08 GB, 230 us (4.7 TB/s: what a workgroup
// costs besides its keys, three rounds of it; eight wavefronts with half the ring each 227); one over 1999, 8 MB, 11.1 us.
//
// S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32: a lane then owns one row throughout (column lane % 16).  The rows
// of the first product's left operand are keys in the order 8 (r / 4) + 4 t + r % 4 for tile t of two, so that a lane's
// eight scores are those of 8 consecutive keys -- which is the operand layout of P in the second product, and the order
// in which the LDS transpose reads deliver V's keys.  K and V blocks go from memory into LDS without registers in between.
//
// A tile's workgroups meet through the workspace (agent_scope.hpp): each leaves its rows' (reference, sum, O), the last one
// to arrive adds them in range order, so the result does not depend on who was last.
constexpr int R16 = 16, R16_WAVES = 4, R16_NT = 64 * R16_WAVES, R16_BK = 32, R16_WINDOW = 256;
constexpr int R16_MIN_BLOCKS = 8;  // blocks of a workgroup below which keys are not cut further: two per wavefront (1999 keys: 12.0 us; with one or four 13.3, 12.2)
template <int D, bool F8> struct SeqGeom {
    static_assert(D == 64 || D == 128, "head dim");
    static constexpr int ES = F8 ? 1 : 2, ROW = D * ES, CPR = ROW / 16, KPI = 64 / CPR;  // bytes and 16-byte chunks of a row, keys of an LDS-DMA instruction
    static constexpr int DMAS = 32 / KPI;           // instructions of a block of 32 keys, 1 KB each
    static constexpr int KS = D / 32, DT = D / 16;  // 32-wide slices of the head dim, 16-wide tiles of the output
    // Bank conflicts.  A K read's 16 lanes go through keys that differ in bits {0, 1, 3, 4}, one chunk each; a V read's 32 lanes through keys
    // that differ in bits {0, 1, 3}, two chunks each (16-bit), or {0, 1, 2, 3}, a chunk each (8-bit).  Keys of one instruction are told
    // apart by an XOR on the chunk index (on the source side), instructions by padding between them; the XOR stays below the bits that
    // step along the head dim in K, so one address per lane serves all of K's fragments, and VB of them V's.
    static constexpr int PADDED_K = 1024 + 32, PADDED_V = 1024 + 64;
    static constexpr int BLOCK_K = DMAS * PADDED_K, BLOCK_V = DMAS * PADDED_V;  // 32 keys
    static __device__ __forceinline__ int kswz(int key) { return ROW == 256 ? key & 3 : ROW == 128 ? (key >> 1) & 1 : (key >> 3) & 1; }
    static __device__ __forceinline__ int vswz(int key) {
        if (F8) return ROW == 128 ? (key >> 1) & 3 : (key >> 2) & 3;
        return (ROW == 256 ? key & 3 : (key >> 1) & 1) << 1;
    }
    // K fragment q = 2 ks + t: 16 keys of tile t, 32 of the head dim
    static constexpr int KF = 2 * KS, K_STEP = 32 * ES, K_TILE = KPI == 4 ? PADDED_K : 4 * ROW;
    static __device__ __forceinline__ int k_lane(int r, int g) {
        const int key = 8 * (r >> 2) + (r & 3);
        return key / KPI * PADDED_K + key % KPI * ROW + (((F8 ? g >> 1 : g) ^ kswz(key)) << 4) + (F8 ? (g & 1) * 8 : 0);
    }
    // V fragment j: 32 keys, 16 of the head dim, in VR transpose reads
    static constexpr int VR = F8 ? 1 : 2, VB = F8 || D == 128 ? 4 : 2, V_STEP = VB * (F8 ? 16 : 32), V_HALF = KPI == 4 ? PADDED_V : 4 * ROW;
    static __device__ __forceinline__ int v_lane(int r, int g, int b) {
        const int key = 8 * g + (F8 ? r >> 1 : r >> 2);
        return key / KPI * PADDED_V + key % KPI * ROW + (((F8 ? b : 2 * b + ((r >> 1) & 1)) ^ vswz(key)) << 4) + (r & 1) * 8;
    }
};
template <int D, bool F8> struct R16Geom : SeqGeom<D, F8> {
    typedef SeqGeom<D, F8> S;
    static constexpr int RING = S::DMAS == 8 ? 2 : 4;        // blocks of K and of V in a wavefront's ring
    static constexpr int BLOCK = S::BLOCK_K + S::BLOCK_V, WAVE = RING * BLOCK;
    static constexpr int LINE = D + 4;                       // floats of a row's (reference, sum, -, -, O)
    static constexpr int MERGE = R16_WAVES * R16 * LINE * 4;
    static constexpr int WINDOW_AT = R16_WAVES * WAVE > MERGE ? R16_WAVES * WAVE : MERGE;
    static constexpr int LDS = WINDOW_AT + R16_WAVES * R16_WINDOW * 4 + 16;
};
// How far a score may exceed the exponent reference of its row before the reference moves (as a power of two), and how far above the
// largest score a new reference is put.  In bf16 by as much: P is at most one, so the sums over the keys reach no further than
// the sum of the values themselves, which may be as large as f32 holds.  f16 keeps few digits of a P below 2^-14, so there P reaches
// up to 2^12 instead; its values are below 2^16, and the sums far from f32's end.  Scores that rise by 2^12 over a row's first are
// rare, and a move of the reference is what a step costs.
template <int CK> struct Slack {
    static constexpr float SLACK = 12.f, LIFT = CK == mfma::CK_F16 ? 0.f : SLACK;
};
// The reference of a row without a key yet.  (Finite, so that a score that is masked, -infinity, is 2^-infinity = 0 of it.)
constexpr float NO_KEY = -__FLT_MAX__;
// c = scale log2 e, kept normal: a masked score times c stays -infinity
__device__ __forceinline__ float exponent_scale(float c) { return c < __FLT_MIN__ ? __FLT_MIN__ : c; }
// 1.0 in every element: the row sums are one more tile of the second product, over the P that it multiplies (which is rounded,
// so that the weights sum to one), and cost no vector instruction and no exchange between a row's lanes
template <int CK> __device__ __forceinline__ u32x4_t ones() {
    const uint32_t w = CK == mfma::CK_BF16 ? 0x3F803F80u : 0x3C003C00u;
    return u32x4_t{w, w, w, w};
}

template <int CK, int D, bool PAGED, bool F8>
__global__ __launch_bounds__(R16_NT) void seq_attention_r16_kernel(const uint16_t *__restrict__ Q, const char *__restrict__ K,
                                                                   const char *__restrict__ V, uint16_t *__restrict__ O, DevSeq a,
                                                                   float *ws, unsigned ws_bytes, int *arrival) {
    typedef R16Geom<D, F8> G;
    typedef Compute<CK> Cmp;
    typedef typename Cmp::acc_t acc_t;
    constexpr bool F16 = CK == mfma::CK_F16;
    HODU_DYNAMIC_LDS(smem);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.kv_heads;
    SeqTile f;
    const int tile = blockIdx.x / a.kv_heads;
    if (!(a.batch <= 64 ? find_tile_long_first<R16, PAGED>(a, tile, f) : find_tile<R16, PAGED>(a, tile, f))) return;
    const int row0 = f.row0, q0 = f.q0, n = f.n, m = f.m, rows = n * a.group;

    // the lane's row; rows past the sequence's last repeat it and are not stored
    const int rr = row0 + r < rows ? row0 + r : rows - 1;
    const int tok = quot(rr, a.by_group), head = kvh * a.group + rr - tok * a.group;
    const int open = a.causal ? attended(tok, n, m) : m;  // keys the row attends, <= 0: none
    const int last_tok = quot(row0 + R16 - 1 < rows ? row0 + R16 - 1 : rows - 1, a.by_group), first_tok = quot(row0, a.by_group);
    const int keys = a.causal ? attended(last_tok, n, m) : m;          // keys the tile needs
    const int all_open = a.causal ? attended(first_tok, n, m) : m;     // keys below this are open to every row
    const int blocks = keys > 0 ? (keys + R16_BK - 1) / R16_BK : 0;
    // the tile's workgroups: as many as the launch has for it and the keys are worth
    const int worth = (blocks + R16_MIN_BLOCKS - 1) / R16_MIN_BLOCKS;
    const int splits = worth < 1 ? 1 : worth < (int)gridDim.y ? worth : (int)gridDim.y;
    const int split = blockIdx.y;
    if (split >= splits) return;
    const int blk0 = (int)((long)blocks * (split * R16_WAVES + wave) / (splits * R16_WAVES)), blk1 = (int)((long)blocks * (split * R16_WAVES + wave + 1) / (splits * R16_WAVES));

    u32x4_t qf[G::KS];
#pragma unroll
    for (int ks = 0; ks < G::KS; ks++)
        qf[ks] = *reinterpret_cast<const u32x4_t *>(Q + (q0 + tok) * a.q_token + head * a.q_head + 32 * ks + 8 * g);
    const float c = exponent_scale(a.scale_log2e * (F8 ? a.k_scale[kvh] : 1.f));
    const float v_scale = F8 ? a.v_scale[kvh] : 1.f;

    char *ring = smem + wave * G::WAVE;
    const unsigned ring0 = (unsigned)(uintptr_t)ring;
    const char *kbase = K + kvh * a.kc.head, *vbase = V + kvh * a.vc.head;
    int *window = reinterpret_cast<int *>(smem + G::WINDOW_AT) + wave * R16_WINDOW;  // the wavefront's next table entries
    int window0 = 0;
    [[maybe_unused]] auto fill_window = [&](int from) __attribute__((always_inline)) {
        const int cols = quot(keys - 1, a.page) + 1;
        mfma::wave_lds_fence();
#pragma unroll
        for (int i = 0; i < R16_WINDOW / 64; i++) {
            const int col = from + i * 64 + lane, pg = a.table[(long)f.b * a.width + (col < cols ? col : cols - 1)];
            window[i * 64 + lane] = pg < 0 ? 0 : pg < a.n_pages ? pg : a.n_pages - 1;
        }
        window0 = from;
        mfma::wave_lds_fence();
    };
    auto issue = [&](int blk, int slot) __attribute__((always_inline)) {
        if constexpr (PAGED) {
            const int last = (blk + 1) * R16_BK < keys ? (blk + 1) * R16_BK - 1 : keys - 1;
            if (quot(last, a.page) - window0 >= R16_WINDOW) fill_window(quot(blk * R16_BK, a.page));
        }
#pragma unroll
        for (int i = 0; i < G::DMAS; i++) {
            const int kk = i * G::KPI + lane / G::CPR;  // the lane's key of this instruction
            int key = blk * R16_BK + kk;
            key = key < keys ? key : keys - 1;  // behind the last key: that one again, masked below
            long ko, vo;
            if constexpr (PAGED) {
                const int col = quot(key, a.page), in = key - col * a.page.d, pg = window[col - window0];
                ko = pg * a.kc.page + in * a.kc.token;
                vo = pg * a.vc.page + in * a.vc.token;
            } else {
                ko = (f.k0 + key) * a.kc.token;
                vo = (f.k0 + key) * a.vc.token;
            }
            const int at = lane % G::CPR;
            const unsigned to = ring0 + slot * G::BLOCK;
            mfma::dma16_raw(kbase + ko + ((at ^ G::kswz(kk)) << 4), __builtin_amdgcn_readfirstlane(to + i * G::PADDED_K));
            mfma::dma16_raw(vbase + vo + ((at ^ G::vswz(kk)) << 4), __builtin_amdgcn_readfirstlane(to + G::BLOCK_K + i * G::PADDED_V));
        }
    };

    acc_t o[G::DT + 1];  // the last tile: the row sums
    // What the remainders of P give is summed apart from what P gives: of an infinite value P makes an infinity, a remainder may make its
    // opposite or, where it is zero, a NaN.  (8-bit values have no infinity.)
    constexpr bool APART = !F8;
    acc_t o_rest[APART ? G::DT : 1];
#pragma unroll
    for (int j = 0; j <= G::DT; j++) o[j] = acc_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < (APART ? G::DT : 1); j++) o_rest[j] = acc_t{0.f, 0.f, 0.f, 0.f};
    const u32x4_t one = ones<CK>();
    const int k_lane = G::k_lane(r, g);
    int v_lane[G::VB];
#pragma unroll
    for (int b = 0; b < G::VB; b++) v_lane[b] = G::v_lane(r, g, b);
    // The reference of the lane's row is a score, the largest when it was last moved; p = 2^(c (s - reference) - LIFT).  The difference is
    // taken of the scores themselves, where it is exact if they are close, however large they are.
    constexpr float SLACK = Slack<CK>::SLACK, LIFT = Slack<CK>::LIFT;
    float ref = NO_KEY;
    if (blk0 < blk1) {
        if constexpr (PAGED) fill_window(quot(blk0 * R16_BK, a.page));
        // (pinned: these loads have returned before the ones are issued that the compiler does not know of)
#pragma unroll
        for (int ks = 0; ks < G::KS; ks++) mfma::pin_vector(qf[ks]);
#pragma unroll
        for (int s = 0; s < G::RING; s++)
            if (blk0 + s < blk1) issue(blk0 + s, s);
    }
    int slot = 0;
    for (int blk = blk0; blk < blk1; blk++) {
        // this block has landed, up to RING - 1 later ones may be in flight
        const int later = blk1 - 1 - blk;
        if (later >= G::RING - 1) __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0((G::RING - 1) * 2 * G::DMAS));
        else if (G::RING > 2 && later == 2) __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(2 * 2 * G::DMAS));
        else if (G::RING > 2 && later == 1) __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(2 * G::DMAS));
        else __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(0));
        mfma::wave_lds_fence();
        char *kl = ring + slot * G::BLOCK, *vl = kl + G::BLOCK_K;
        if constexpr (APART) {
            // the copies of the last key, which P is zero of: an infinite value times zero would be a NaN
            if ((blk + 1) * R16_BK > keys) {
#pragma unroll
                for (int i = 0; i < G::DMAS; i++)
                    if (blk * R16_BK + i * G::KPI + lane / G::CPR >= keys)
                        *reinterpret_cast<u32x4_t *>(vl + i * G::PADDED_V + lane * 16) = u32x4_t{0, 0, 0, 0};
                __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(63));
                mfma::wave_lds_fence();
            }
        }

        acc_t s[2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            s[t] = acc_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < G::KS; ks++) {
                const int at = k_lane + ks * G::K_STEP + t * G::K_TILE;
                u32x4_t kf;
                if constexpr (F8) kf = widen8<CK>(lds_get64(kl, at));
                else kf = lds_get(kl, at);
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
        float top = sv[0];
#pragma unroll
        for (int e = 1; e < 8; e++) top = __builtin_fmaxf(top, sv[e]);
        if (__builtin_amdgcn_ballot_w64(c * (top - ref) > SLACK) != 0) {
            top = __builtin_fmaxf(top, __shfl_xor(top, 16));
            top = __builtin_fmaxf(top, __shfl_xor(top, 32));
            const float next = c * (top - ref) > SLACK ? top : ref;
            const float keep = __builtin_amdgcn_exp2f(c * (ref - next));
            ref = next;
            if (blk != blk0)  // (the first block's sums are zero)
#pragma unroll
                for (int j = 0; j <= G::DT; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        o[j][e] *= keep;
                        if constexpr (APART)
                            if (j < G::DT) o_rest[j][e] *= keep;
                    }
        }
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e] - ref, c, -LIFT));
        const u32x4_t pf = {pack2<CK>(p[0], p[1]), pack2<CK>(p[2], p[3]), pack2<CK>(p[4], p[5]), pack2<CK>(p[6], p[7])};
        // What P's rounding left is multiplied too, as a second operand: a single token's output is then as exact as its own rounding (the
        // matrix instructions are not the bound here; with P rounded once the error was 1.4 times that).
        float rest[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint16_t w = (uint16_t)(pf[e >> 1] >> (16 * (e & 1)));
            rest[e] = p[e] - (F16 ? f16_bits_to_f32(w) : bf16_bits_to_f32(w));
        }
        const u32x4_t pr = {pack2<CK>(rest[0], rest[1]), pack2<CK>(rest[2], rest[3]), pack2<CK>(rest[4], rest[5]), pack2<CK>(rest[6], rest[7])};
        Cmp::mma(one, pf, o[G::DT]);
        Cmp::mma(one, pr, o[G::DT]);
#pragma unroll
        for (int j = 0; j < G::DT; j++) {
            const int at = v_lane[j % G::VB] + j / G::VB * G::V_STEP;
            u32x4_t vf;
            if constexpr (F8) {
                vf = widen8<CK>(lds_get_tr<1>(vl, at));
            } else {
                const u32x2_t lo = lds_get_tr<2>(vl, at), hi = lds_get_tr<2>(vl, at + G::V_HALF);
                vf = u32x4_t{lo.x, lo.y, hi.x, hi.y};
            }
            Cmp::mma(vf, pf, o[j]);
            if constexpr (APART) Cmp::mma(vf, pr, o_rest[j]);
            else Cmp::mma(vf, pr, o[j]);
        }
        if (blk + G::RING < blk1) {
            // the block's reads have been answered before its slot's next loads are issued
            __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(63));
            mfma::wave_lds_fence();
            issue(blk + G::RING, slot);
        }
        slot = slot + 1 < G::RING ? slot + 1 : 0;
    }

    if constexpr (APART) {
        float size = 0.f;
#pragma unroll
        for (int j = 0; j < G::DT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) size = __builtin_fmaxf(size, __builtin_fabsf(o[j][e]));
        const bool finite = __builtin_amdgcn_ballot_w64(size == INFINITY) == 0;
#pragma unroll
        for (int j = 0; j < G::DT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (finite || __builtin_fabsf(o[j][e]) != INFINITY) o[j][e] += o_rest[j][e];
    }
    // ---- the four wavefronts meet: per wavefront and row (reference, sum, -, -, O) ----
    __syncthreads();
    float *mg = reinterpret_cast<float *>(smem);
    {
        float *mine = mg + (wave * R16 + r) * G::LINE;
        if (g == 0) {
            mine[0] = ref;
            mine[1] = o[G::DT][0];
        }
#pragma unroll
        for (int j = 0; j < G::DT; j++) *reinterpret_cast<f32x4_t *>(mine + 4 + 16 * j + 4 * g) = f32x4_t{o[j][0], o[j][1], o[j][2], o[j][3]};
    }
    __syncthreads();
    constexpr int PARTS = R16_NT / R16, PER = D / PARTS;  // threads of a row, elements of each
    const int row = tid / PARTS, part = tid % PARTS;
    float all = NO_KEY, l = 0.f, x[PER];
#pragma unroll
    for (int i = 0; i < R16_WAVES; i++) all = __builtin_fmaxf(all, mg[(i * R16 + row) * G::LINE]);
#pragma unroll
    for (int e = 0; e < PER; e++) x[e] = 0.f;
#pragma unroll
    for (int i = 0; i < R16_WAVES; i++) {
        const float *line = mg + (i * R16 + row) * G::LINE;
        const float w = __builtin_amdgcn_exp2f(c * (line[0] - all));
        l += line[1] * w;
#pragma unroll
        for (int e = 0; e < PER; e++) x[e] += line[4 + part * PER + e] * w;
    }
    if (splits > 1) {
        const __amdgpu_buffer_rsrc_t buf = agent_buffer(ws, ws_bytes);
        const unsigned tile_at = blockIdx.x * gridDim.y * R16 * G::LINE * 4, mine = tile_at + (split * R16 + row) * G::LINE * 4;
        if (part == 0) store16_agent(buf, mine, f32x4_t{all, l, 0.f, 0.f});
#pragma unroll
        for (int e = 0; e < PER; e += 4) store16_agent(buf, mine + (4 + part * PER + e) * 4, f32x4_t{x[e], x[e + 1], x[e + 2], x[e + 3]});
        int *flag = reinterpret_cast<int *>(smem + G::WINDOW_AT + R16_WAVES * R16_WINDOW * 4);
        if (!arrive_and_check_last(arrival + blockIdx.x, splits, flag, tid)) return;
        // (eight ranges' loads in flight at once: each is a trip to memory)
        all = NO_KEY;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < PER; e++) x[e] = 0.f;
        for (int i0 = 0; i0 < splits; i0 += 8) {
            f32x4_t h[8], y[8][PER / 4];
            float top = all;
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const unsigned at = tile_at + ((i0 + u < splits ? i0 + u : splits - 1) * R16 + row) * G::LINE * 4;
                h[u] = load16_agent<f32x4_t>(buf, at);
#pragma unroll
                for (int e = 0; e < PER / 4; e++) y[u][e] = load16_agent<f32x4_t>(buf, at + (4 + part * PER + 4 * e) * 4);
            }
#pragma unroll
            for (int u = 0; u < 8; u++) top = __builtin_fmaxf(top, h[u].x);
            const float f = __builtin_amdgcn_exp2f(c * (all - top));
            all = top;
            l *= f;
#pragma unroll
            for (int e = 0; e < PER; e++) x[e] *= f;
#pragma unroll
            for (int u = 0; u < 8; u++) {
                if (i0 + u >= splits) break;
                const float w = __builtin_amdgcn_exp2f(c * (h[u].x - all));
                l += h[u].y * w;
#pragma unroll
                for (int e = 0; e < PER; e++) x[e] += y[u][e / 4][e % 4] * w;
            }
        }
        arrival_reset(arrival + blockIdx.x, tid);
    }
    if (row0 + row >= rows) return;
    const float inv = l == 0.f ? 0.f : v_scale / l;  // a row without keys: l = 0, and zero is what it gives
    const int wtok = quot(row0 + row, a.by_group), whead = kvh * a.group + row0 + row - wtok * a.group;
    uint32_t out[PER / 2];
#pragma unroll
    for (int e = 0; e < PER; e += 2) out[e / 2] = pack2<CK>(x[e] * inv, x[e + 1] * inv);
    uint16_t *dst = O + ((long)(q0 + wtok) * a.heads + whead) * D + part * PER;
    if constexpr (PER >= 8)
#pragma unroll
        for (int e = 0; e < PER / 2; e += 4) *reinterpret_cast<u32x4_t *>(dst + 2 * e) = u32x4_t{out[e], out[e + 1], out[e + 2], out[e + 3]};
    else *reinterpret_cast<u32x2_t *>(dst) = u32x2_t{out[0], out[1]};
}

// ---- tiles of 128, 192 or 256 rows, one wavefront per SIMD ---------------------------------------------------------------
// The matrix cores bound a long prompt: 4 D flops per (row, key) pair against 2 D / rows bytes.  Four wavefronts own 16 RT
// rows each (RT = 2, 3 or 4 tiles of 16) and walk all keys of the tile, 64 to a stage of the LDS ring, 32 to a step, with the layouts of the
// kernel above.  A fragment of K or V read from LDS feeds RT matrix instructions, which is what keeps LDS from being the bound
// (128 bytes a cycle: a fragment per 2 RT cycles of each SIMD; the instruction takes 16).
// Measured, bf16, causal, 32 query and 8 key / value heads of 128: 8192 tokens 544 us (1010 TFLOP/s; a matrix product of 8192^3 runs
// at 1210); 16 prompts of up to 2048 tokens 392 us (626: a workgroup costs some 10 us besides its stages of 1.5 us, and a tile of
// those has 10 of them); four chunks of 512 tokens over up to 8192 285 us (758).
//
// P is rounded to the type for the second product, and the row sum is taken of it as rounded: the output is off by 1.3 to 1.4 times
// what its own rounding costs.  What the rounding leaves could be multiplied too, as the kernel above does where memory is the bound;
// here it would be 27 more matrix instructions to a step of 51 (head dim 128, three tiles), and they are the bound.
//
// A wavefront issues in order, an instruction every 4 cycles, and a matrix instruction runs for 16: the exponentials have
// to stand BETWEEN the matrix instructions.  So a step holds three independent pieces of work -- scores of step i + 1,
// exponentials of step i, P V of step i - 1 -- written out as one sequence of chunks, a matrix instruction and
// a share of the vector work and LDS reads in each, which the compiler may not reorder across (sched_barrier, and the empty
// statements that pin a chunk's results to it).
//
// The exponent reference of a row is an integer E, ceil(c max) + LIFT when it was last set, c = scale log2 e; p = 2^(c s - E).  It moves only
// when a score reaches c s > E + SLACK - LIFT, which the lanes find out without talking to each other (any lane's own maximum); then the
// row's lanes agree on the new one and O, the row sum and the P not yet multiplied are rescaled -- by a power of two, exactly.
// That takes |c s| far below 2^24, where E and c s are told apart to less than one.  A wavefront that meets larger ones (its first
// scores, or one that moves a reference) turns careful: its references become scores, p = 2^(c (s - reference) - LIFT) as in
// the kernel above, where a difference is exact if the scores are close, and it takes the slow step from there on.  In the
// loops that would be an instruction per exponential between matrix instructions that are 16 cycles long already.
// Row tiles per wavefront: 3 at head dim 128 (O, q, two steps' scores and P are 84 registers a tile; with 4 the allocator runs out),
// 4 at 64.
template <int D> constexpr int W_TILES = D == 128 ? 3 : 4;
constexpr int W_NT = 256, W_BK = 64, W_RING = 4, W_WINDOW = 2048, W_MIN_STAGES = 8;  // (the ring: stages of K and of V)
template <int D, bool F8, bool PAGED> struct WGeom : SeqGeom<D, F8> {
    typedef SeqGeom<D, F8> S;
    static constexpr int NI = 2 * S::DMAS / 4;               // LDS-DMA instructions per stage of K (of V) and wavefront
    static constexpr int V_AT = W_RING * 2 * S::BLOCK_K, TABLE_AT = V_AT + W_RING * 2 * S::BLOCK_V;
    static constexpr int LDS = TABLE_AT + (PAGED ? W_WINDOW * 4 : 0);
};

// lds_get_tr of an address that stays one of LDS for the compiler, which then adds its constant parts in the instruction
typedef char __attribute__((address_space(3))) * lds_bytes_t;
template <int SB> __device__ __forceinline__ u32x2_t lds_transpose(lds_bytes_t at) {
    if constexpr (SB == 2) {
        typedef short s16x4_t __attribute__((ext_vector_type(4)));
        typedef s16x4_t __attribute__((address_space(3))) * lds_ptr_t;
        return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr_t)at));
    } else {
        typedef int i32x2_t __attribute__((ext_vector_type(2)));
        typedef i32x2_t __attribute__((address_space(3))) * lds_ptr_t;
        return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_ptr_t)at));
    }
}

template <int CK, int D, bool PAGED, bool F8, int RT>
__global__ __launch_bounds__(W_NT, 1) void seq_attention_wide_kernel(const uint16_t *__restrict__ Q, const char *__restrict__ K,
                                                                     const char *__restrict__ V, uint16_t *__restrict__ O, DevSeq a,
                                                                     float *ws, unsigned ws_bytes, int *arrival) {
    typedef WGeom<D, F8, PAGED> G;
    typedef Compute<CK> Cmp;
    typedef typename Cmp::acc_t acc_t;
    constexpr int KS = G::KS, DT = G::DT, BM = 64 * RT;
    constexpr bool F16 = CK == mfma::CK_F16;
    HODU_DYNAMIC_LDS(smem);
    const unsigned lds0 = (unsigned)(uintptr_t)smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.kv_heads;
    SeqTile f;
    const int tile = blockIdx.x / a.kv_heads;
    if (!(a.batch <= 64 ? find_tile_long_first<BM, PAGED>(a, tile, f) : find_tile<BM, PAGED>(a, tile, f))) return;
    const int b = f.b, row0 = f.row0, q0 = f.q0, n = f.n, k0 = f.k0, m = f.m, rows = n * a.group;
    // the lane's rows, one per tile; rows past the sequence's last repeat it and are not stored
    int open[RT];
    u32x4_t qf[RT][KS];
    const int wrow0 = row0 + wave * 16 * RT;
#pragma unroll
    for (int x = 0; x < RT; x++) {
        const int row = wrow0 + 16 * x + r, rr = row < rows ? row : rows - 1;
        const int tok = quot(rr, a.by_group), head = kvh * a.group + rr - tok * a.group;
        open[x] = a.causal ? attended(tok, n, m) : m;  // keys the row attends, <= 0: none
        const uint16_t *q = Q + (q0 + tok) * a.q_token + head * a.q_head;
#pragma unroll
        for (int ks = 0; ks < KS; ks++) qf[x][ks] = *reinterpret_cast<const u32x4_t *>(q + 32 * ks + 8 * g);
    }
    const float c = exponent_scale(a.scale_log2e * (F8 ? a.k_scale[kvh] : 1.f));
    auto last_row = [&](int i) { return i < rows ? i : rows - 1; };
    const int keys_any = a.causal ? attended(quot(last_row(row0 + BM - 1), a.by_group), n, m) : m;  // keys the tile needs
    int keys = keys_any > 0 ? keys_any : 0;
    int wave_keys = a.causal ? attended(quot(last_row(wrow0 + 16 * RT - 1), a.by_group), n, m) : m;  // ... the wavefront needs
    int all_open = a.causal ? attended(quot(last_row(wrow0), a.by_group), n, m) : m;  // keys below this are open to all its rows
    int stages = (keys + W_BK - 1) / W_BK;
    // few tiles over a long cache: this workgroup's range of the keys, and everything from here on counts from its first one
    int from = 0, splits = 1;
    if constexpr (PAGED) {
        const int worth = stages / W_MIN_STAGES, split = blockIdx.y;
        splits = worth < 1 ? 1 : worth < (int)gridDim.y ? worth : (int)gridDim.y;
        if (split >= splits) return;
        if (splits > 1) {
            const int s0 = stages * split / splits, s1 = stages * (split + 1) / splits;
            from = s0 * W_BK;
            stages = s1 - s0;
            keys = (keys < s1 * W_BK ? keys : s1 * W_BK) - from;
            wave_keys = wave_keys - from < keys ? wave_keys - from : keys;
            all_open = all_open - from < keys ? all_open - from : keys;
#pragma unroll
            for (int x = 0; x < RT; x++) open[x] -= from;
        }
    }
    const int steps = wave_keys > 0 && wrow0 < rows ? (wave_keys + 31) / 32 : 0;  // of 32 keys, that the wavefront needs

    // ---- memory -> LDS: instruction i of a block fills 1 KB, KPI keys; a wavefront issues NI of them for K and for V ----
    const char *kbase = K + kvh * a.kc.head, *vbase = V + kvh * a.vc.head;
    int *window = reinterpret_cast<int *>(smem + G::TABLE_AT);
    int window0 = 0;  // first table column in the window
    [[maybe_unused]] auto fill_window = [&](int col0) __attribute__((always_inline)) {
        const int cols = quot(from + keys - 1, a.page) + 1;
        int i = tid;
        mfma::pin_vector(i);  // (or the compiler keeps addresses made from it in registers throughout the kernel)
        for (; i < W_WINDOW && col0 + i < cols; i += W_NT) {
            const int pg = a.table[(long)b * a.width + col0 + i];
            window[i] = pg < 0 ? 0 : pg < a.n_pages ? pg : a.n_pages - 1;
        }
        window0 = col0;
    };
    // a lane's source within a stage of packed keys (the token stride is below 2^25 bytes: the host sees to it)
    unsigned in_stage[2][G::NI];
#pragma unroll
    for (int p = 0; p < G::NI; p++) {
        const int kk = (wave * G::NI + p) * G::KPI + lane / G::CPR;
        in_stage[0][p] = kk * (unsigned)a.kc.token + (((lane % G::CPR) ^ G::kswz(kk & 31)) << 4);
        in_stage[1][p] = kk * (unsigned)a.vc.token + (((lane % G::CPR) ^ G::vswz(kk & 31)) << 4);
    }
    // The same of a paged cache: page and token within it of the lane's key of each instruction.  K is loaded a stage ahead of V, so a
    // key is looked up once, in the stage before its K is issued (between the matrix instructions), and what K used V uses next.
    [[maybe_unused]] int k_page[G::NI], k_in[G::NI], v_page[G::NI], v_in[G::NI];
    auto look_up = [&](int stage, int p) __attribute__((always_inline)) {
        int key = stage * W_BK + (wave * G::NI + p) * G::KPI + lane / G::CPR;
        key = from + (key < keys ? key : keys - 1);  // behind the last key: that one again, masked below
        const int col = quot(key, a.page);
        k_page[p] = window[col - window0];
        k_in[p] = key - col * a.page.d;
    };
    auto pass_on = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < G::NI; p++) v_page[p] = k_page[p], v_in[p] = k_in[p];
    };
    auto issue = [&](int stage, bool is_v) __attribute__((always_inline)) {
        const PagedSide &side = is_v ? a.vc : a.kc;
        const char *base = is_v ? vbase : kbase;
        const unsigned padded = is_v ? G::PADDED_V : G::PADDED_K;
        // (a stage is two blocks of 32 keys, the ring eight)
        const unsigned to = lds0 + (is_v ? G::V_AT : 0) + (stage & (W_RING - 1)) * 2 * (is_v ? G::BLOCK_V : G::BLOCK_K) + wave * G::NI * padded;
        if (!PAGED && (stage + 1) * W_BK <= keys) {
            const char *keys0 = base + (long)(k0 + stage * W_BK) * side.token;
#pragma unroll
            for (int p = 0; p < G::NI; p++) mfma::dma16_sbase(keys0, in_stage[is_v][p], __builtin_amdgcn_readfirstlane(to + p * padded));
            return;
        }
#pragma unroll
        for (int p = 0; p < G::NI; p++) {
            const int kk = (wave * G::NI + p) * G::KPI + lane / G::CPR;
            long off;
            if constexpr (PAGED) {
                // (32-bit strides, and a page's tokens are within 2^32 bytes: the host sees to it)
                off = (unsigned long)(unsigned)(is_v ? v_page[p] : k_page[p]) * (unsigned)side.page + (unsigned)(is_v ? v_in[p] : k_in[p]) * (unsigned)side.token;
            } else {
                int key = stage * W_BK + kk;
                key = key < keys ? key : keys - 1;  // behind the last key: that one again, masked below
                off = (k0 + key) * side.token;
            }
            const int chunk = (lane % G::CPR) ^ (is_v ? G::vswz(kk & 31) : G::kswz(kk & 31));
            mfma::dma16_raw(base + off + (chunk << 4), __builtin_amdgcn_readfirstlane(to + p * padded));
        }
    };

    acc_t o[RT][DT + 1];           // the last tile: the row sums
    float e_ref[RT], top[RT];      // exponent reference, the lane's largest new score
    float lowest = -INFINITY;
    mfma::pin_vector(lowest);  // (one instruction for a row's first two scores: as a constant it would vanish, and leave three)
    u32x4_t one = ones<CK>();
    mfma::pin_vector(one);  // (or the compiler makes it anew in every step)
#pragma unroll
    for (int x = 0; x < RT; x++) {
#pragma unroll
        for (int j = 0; j <= DT; j++) o[x][j] = acc_t{0.f, 0.f, 0.f, 0.f};
        e_ref[x] = NO_KEY;
    }

    constexpr int KF = G::KF, VR = G::VR;
    typedef typename std::conditional<F8, u32x2_t, u32x4_t>::type raw_t;  // (8-bit: raw bytes, widened at their use)
    raw_t kf[KF];
    u32x2_t vf[DT * VR];
    const int k_lane = G::k_lane(r, g);
    int v_lane[G::VB];
    lds_bytes_t v_from[G::VB];
#pragma unroll
    for (int b2 = 0; b2 < G::VB; b2++) v_lane[b2] = G::V_AT + G::v_lane(r, g, b2);
    auto read_k = [&](int q, int at) __attribute__((always_inline)) {
        const int from = k_lane + at + (q >> 1) * G::K_STEP + (q & 1) * G::K_TILE;
        if constexpr (F8) kf[q] = lds_get64(smem, from);
        else kf[q] = lds_get(smem, from);
    };
    auto k_operand = [&](int q) __attribute__((always_inline)) -> u32x4_t {
        if constexpr (F8) return widen8<CK>(kf[q]);
        else return kf[q];
    };
    auto read_v = [&](int q, int at) __attribute__((always_inline)) {
        const int j = q / VR;
        if (q % VR == 0 && j < G::VB) {
            v_from[j] = (lds_bytes_t)smem + v_lane[j] + at;
            mfma::pin_vector(v_from[j]);  // (one register, and what is added to it below an immediate)
        }
        vf[q] = lds_transpose<F8 ? 1 : 2>(v_from[j % G::VB] + j / G::VB * G::V_STEP + q % VR * G::V_HALF);
    };
    auto v_operand = [&](int j) __attribute__((always_inline)) -> u32x4_t {
        if constexpr (F8) return widen8<CK>(vf[j]);
        else return u32x4_t{vf[2 * j].x, vf[2 * j].y, vf[2 * j + 1].x, vf[2 * j + 1].y};
    };
    // scores of step i beyond what a row attends; the lane's keys are 8 g + 4 t + e
    auto mask = [&](acc_t (&sc)[RT][2], int i) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const int left = open[x] - (i * 32 + 8 * g);
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) sc[x][t][e] = 4 * t + e < left ? sc[x][t][e] : -INFINITY;
        }
    };
    auto largest = [&](const acc_t (&sc)[RT][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < RT; x++) {
            top[x] = sc[x][0][0];
#pragma unroll
            for (int e = 1; e < 8; e++) top[x] = __builtin_fmaxf(top[x], sc[x][e >> 2][e & 3]);
        }
    };
    constexpr float SLACK = Slack<CK>::SLACK, LIFT = Slack<CK>::LIFT;
    int careful = 0;  // 1: the wavefront's references are scores (see above)
    constexpr float MOST = 0x1p22f;
    // the row's largest new score, the same in its four lanes
    auto row_top = [&](int x) __attribute__((always_inline)) {
        const float most = __builtin_fmaxf(top[x], __shfl_xor(top[x], 16));
        return __builtin_fmaxf(most, __shfl_xor(most, 32));
    };
    // Moves the references of the rows whose new scores exceed them by too much (rare: some lane saw one); pc: the P that is
    // still to be multiplied
    auto move_references = [&](u32x4_t (&pc)[RT]) __attribute__((always_inline)) {
        mfma::mfma_results_settle();
        __builtin_amdgcn_sched_barrier(0);
        float most[RT], f[RT];
        bool far = false;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            most[x] = row_top(x);
            f[x] = 1.f;
            far |= !(c * most[x] <= MOST) && most[x] > 0.f;  // (only a score that is larger than the reference moves it)
        }
        if (!careful && __builtin_amdgcn_ballot_w64(far) != 0) {
            careful = 1;
#pragma unroll
            for (int x = 0; x < RT; x++)
                if (e_ref[x] != NO_KEY) {
                    const float e = e_ref[x] - LIFT, s = e / c, ref = __builtin_fminf(s, __FLT_MAX__);
                    f[x] = __builtin_amdgcn_exp2f(__builtin_fmaf(-ref, c, e));
                    e_ref[x] = ref;
                }
        }
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const float from = e_ref[x];
            if (careful) {
                if (c * (most[x] - from) > SLACK) e_ref[x] = most[x];
                f[x] *= __builtin_amdgcn_exp2f(c * (from - e_ref[x]));
            } else {
                if (c * most[x] > from + (SLACK - LIFT)) e_ref[x] = ceilf(c * most[x]) + LIFT;
                f[x] = __builtin_amdgcn_exp2f(from - e_ref[x]);
            }
#pragma unroll
            for (int j = 0; j <= DT; j++) mfma::scale4_acc(o[x][j], f[x]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t pw = pc[x][i];
                if constexpr (!F16) pc[x][i] = pack2<CK>(bf16_bits_to_f32((uint16_t)pw) * f[x], bf16_bits_to_f32((uint16_t)(pw >> 16)) * f[x]);
                else pc[x][i] = pack2<CK>(f16_bits_to_f32((uint16_t)pw) * f[x], f16_bits_to_f32((uint16_t)(pw >> 16)) * f[x]);
            }
        }
        mfma::mfma_results_settle();
        __builtin_amdgcn_sched_barrier(0);
    };
    // the first ones: there is nothing to rescale yet.  (The keys that a row attends begin with the first one: a row without a key here has none.)
    auto set_references = [&]() __attribute__((always_inline)) {
        float most[RT];
        bool far = false;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            most[x] = row_top(x);
            far |= most[x] > -INFINITY && !(__builtin_fabsf(c * most[x]) <= MOST);
        }
        careful = __builtin_amdgcn_ballot_w64(far) != 0 ? 1 : 0;
#pragma unroll
        for (int x = 0; x < RT; x++)
            if (most[x] > -INFINITY) e_ref[x] = careful ? most[x] : ceilf(c * most[x]) + LIFT;
    };
    auto some_exceed = [&]() __attribute__((always_inline)) {
        bool up = false;
#pragma unroll
        for (int x = 0; x < RT; x++) up |= c * top[x] > e_ref[x] + (SLACK - LIFT);
        return __builtin_amdgcn_ballot_w64(up) != 0;
    };
    auto some_exceed_scores = [&]() __attribute__((always_inline)) {
        bool up = false;
#pragma unroll
        for (int x = 0; x < RT; x++) up |= c * (top[x] - e_ref[x]) > SLACK;
        return __builtin_amdgcn_ballot_w64(up) != 0;
    };
    // element t (of 8 RT) of a step's exponentials
    float pair;
    auto exponential = [&](auto either, const acc_t (&sc)[RT][2], u32x4_t (&pc)[RT], int t) __attribute__((always_inline)) {
        const int x = t >> 3, e = t & 7;
        float s = sc[x][e >> 2][e & 3], less = e_ref[x];
        if constexpr (decltype(either)::value) {
            s -= careful ? less : 0.f;
            less = careful ? LIFT : less;
        }
        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -less));
        if (e & 1) {
            pc[x][e >> 1] = pack2<CK>(pair, v);
            uint32_t w = pc[x][e >> 1];
            mfma::pin_vector(w);
            pc[x][e >> 1] = w;
        } else {
            pair = v;
            mfma::pin_vector(pair);
        }
    };
    constexpr int NQ = KF * RT, NP = DT * RT, EL = 8 * RT, EVERY = (NQ + NP) / EL;
    static_assert(EVERY * EL == NQ + NP, "the exponentials spread evenly over the matrix instructions");
    // where K and V of step i lie in their rings
    auto k_of = [&](int i) __attribute__((always_inline)) { return (i & (2 * W_RING - 1)) * G::BLOCK_K; };
    auto v_of = [&](int i) __attribute__((always_inline)) { return (i & (2 * W_RING - 1)) * G::BLOCK_V; };
    // Step i: scores of i + 1 (into sn) and the lane's largest of them, exponentials of i (sc, into pc), P V of i - 1 (pp).  A fragment is read AHEAD chunks (16 cycles each) before its first use: the first ones of a step in the step before.
    constexpr int AHEAD = NQ < 10 ? NQ : 10;
    auto first_fragments = [&](int k_block) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < KF; q++)
            if (q * RT < AHEAD) read_k(q, k_block);
    };
    // masked: some row may not attend all of step i + 1
    auto step = [&](auto masked, auto second, int i, const acc_t (&sc)[RT][2], acc_t (&sn)[RT][2], const u32x4_t (&pp)[RT], u32x4_t (&pc)[RT]) __attribute__((always_inline)) {
        const int v_block = v_of(i - 1), k_block = k_of(i + 1), k_next = k_of(i + 2);
        constexpr int FROM = NP / 4, MPC = (EL + NP - FROM - 1) / (NP - FROM);
        static_assert(FROM >= 2 && AHEAD <= NP, "");
#pragma unroll
        for (int t = 0; t < NQ + NP; t++) {
            const int u = t - NQ;  // of the P V instructions
            if (t < NQ) {
                // (The scores' matrix instructions name their registers: the allocator would put the scores where the exponentials
                // cannot read them, 32 copies a step.)
                const int q = t / RT, x = t % RT;
                if (q < 2) mfma::mfma16_first<F16, F8>(k_operand(q), qf[x][q >> 1], sn[x][q & 1]);
                else mfma::mfma16_next<F16, F8>(k_operand(q), qf[x][q >> 1], sn[x][q & 1]);
            } else {
                Cmp::mma(v_operand(u / RT), pp[u % RT], o[u % RT][u / RT]);
                if (u >= NP - RT) Cmp::mma(one, pp[u % RT], o[u % RT][DT]);
            }
            if (t % EVERY == 0) exponential(std::false_type(), sc, pc, t / EVERY);
            const int soon = t + AHEAD;  // the instruction whose fragment is read now, if it is the first to use it
            if (soon < NQ) {
                if (soon % RT == 0) read_k(soon / RT, k_block);
            } else if (soon < NQ + NP) {
                if ((soon - NQ) % RT == 0)
#pragma unroll
                    for (int w = 0; w < VR; w++) read_v((soon - NQ) / RT * VR + w, v_block);
            } else if ((soon - NQ - NP) % RT == 0) {
                read_k((soon - NQ - NP) / RT, k_next);
            }
            // (in the second step of a stage: the keys whose K the next stage issues)
            if constexpr (PAGED && decltype(second)::value)
                if (t % 8 == 1 && t / 8 < G::NI) look_up((i >> 1) + 4, t / 8);
            if (u == FROM) {
                // Here the scores become values that anything but a matrix instruction may use: the compiler, which knows nothing
                // of the wait states behind an instruction it has not chosen, copies them for the loop's exits.  (The last one of
                // them was issued FROM matrix instructions ago: its 4 passes are over.)
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    mfma::pin_vector(sn[x][0]);
                    mfma::pin_vector(sn[x][1]);
                }
                if constexpr (decltype(masked)::value) mask(sn, i + 1);
            }
            if (u >= FROM) {  // the lane's largest new score
#pragma unroll
                for (int w = 0; w < MPC; w++) {
                    const int at = (u - FROM) * MPC + w, x = at >> 3, e = at & 7;
                    if (at < EL) top[x] = __builtin_fmaxf(e == 0 ? lowest : top[x], sn[x][e >> 2][e & 3]);
                }
                const int x = ((u - FROM) * MPC + MPC - 1) >> 3;
                if (x < RT) mfma::pin_vector(top[x]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // the same step one piece after the other with few registers, for the first scores and behind a reference that moved; sc: scores of step i, replaced by
    // those of i + 1; pc: P of step i - 1, replaced by that of i
    auto times_v = [&](int i, const u32x4_t (&pp)[RT]) __attribute__((always_inline)) {
        const int at = v_of(i);
#pragma unroll
        for (int x = 0; x < RT; x++) Cmp::mma(one, pp[x], o[x][DT]);
#pragma unroll
        for (int q = 0; q < DT * VR; q++) read_v(q, at);
#pragma unroll
        for (int j = 0; j < DT; j++)
#pragma unroll
            for (int x = 0; x < RT; x++) Cmp::mma(v_operand(j), pp[x], o[x][j]);
    };
    auto slow_step = [&](int i, acc_t (&sc)[RT][2], u32x4_t (&pc)[RT]) __attribute__((always_inline)) {
        if (i > 0) times_v(i - 1, pc);
        if (i >= 0)
#pragma unroll
            for (int t = 0; t < EL; t++) exponential(std::true_type(), sc, pc, t);
        const int at = k_of(i + 1);
#pragma unroll
        for (int q = 0; q < KF; q++) read_k(q, at);
#pragma unroll
        for (int q = 0; q < KF; q++)
#pragma unroll
            for (int x = 0; x < RT; x++) {
                if (q < 2) sc[x][q & 1] = acc_t{0.f, 0.f, 0.f, 0.f};
                Cmp::mma(k_operand(q), qf[x][q >> 1], sc[x][q & 1]);
            }
        if ((i + 2) * 32 > all_open) mask(sc, i + 1);  // some row does not attend all of step i + 1
        largest(sc);
    };

    if (stages > 0) {
        if constexpr (PAGED) {
            fill_window(quot(from, a.page));
            __syncthreads();
        }
        // step 0 multiplies a P of zeros by what lies where V of the step before it would: zeros too
        for (int i = tid; i < G::BLOCK_V / 16; i += W_NT)
            *reinterpret_cast<u32x4_t *>(smem + G::V_AT + (2 * W_RING - 1) * G::BLOCK_V + i * 16) = u32x4_t{0, 0, 0, 0};
#pragma unroll
        for (int ahead = 0; ahead < 3; ahead++) {
            if constexpr (PAGED)
#pragma unroll
                for (int p = 0; p < G::NI; p++) look_up(ahead, p);
            if (ahead < stages) issue(ahead, false);
            if constexpr (PAGED) pass_on();
            if (ahead < 2 && ahead < stages) issue(ahead, true);
        }
        if constexpr (PAGED)
#pragma unroll
            for (int p = 0; p < G::NI; p++) look_up(3, p);
        __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(0));
        // (pinned, so that the compiler knows on every path into the loop that these loads have returned)
#pragma unroll
        for (int x = 0; x < RT; x++)
#pragma unroll
            for (int ks = 0; ks < KS; ks++) mfma::pin_accumulation(qf[x][ks]);
        __syncthreads();
        int st = 0;
        // may_end: the stage may be the tile's last
        auto begin_stage = [&](auto may_end) __attribute__((always_inline)) {
            // K of stage st + 1 and V of stage st have landed (what was issued at the last stage may be in flight), everybody's;
            // and everybody is done with what this stage's loads overwrite
            if (st > 0 && st + 2 < stages) __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(2 * G::NI));
            else __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(0));
            if constexpr (!F8 && decltype(may_end)::value) {
                // the copies of the last key, which P is zero of: an infinite value times zero would be a NaN.  (Each wavefront its own,
                // which have landed; 8-bit values have no infinity.)
                if ((st + 1) * W_BK > keys) {
                    int l = lane;
                    mfma::pin_vector(l);  // (no address of this is kept in a register elsewhere)
#pragma unroll
                    for (int p = 0; p < G::NI; p++) {
                        const int at = wave * G::NI + p;
                        if (st * W_BK + at * G::KPI + l / G::CPR >= keys)
                            *reinterpret_cast<u32x4_t *>(smem + G::V_AT + (st & (W_RING - 1)) * 2 * G::BLOCK_V + at * G::PADDED_V + l * 16) = u32x4_t{0, 0, 0, 0};
                    }
                    __builtin_amdgcn_s_waitcnt(mfma::waitcnt_vm_lgkm0(0));
                }
            }
            __syncthreads();
            if (st + 2 < stages) issue(st + 2, true);
            if (st + 3 < stages) issue(st + 3, false);
            if constexpr (PAGED) {
                pass_on();
                // the table columns of the keys that are looked up in this stage, K of stage st + 4
                const int hi = from + ((st + 5) * W_BK - 1 < keys ? (st + 5) * W_BK - 1 : keys - 1);
                if (st + 4 < stages && quot(hi, a.page) - window0 >= W_WINDOW) {
                    __syncthreads();  // (everybody has looked up what the window held)
                    fill_window(quot(from + (st + 4) * W_BK, a.page));
                    __syncthreads();
                }
            }
        };
        // Two loops, one for stages whose scores are all open and one that masks, hold nothing but the two steps: a rarely taken
        // block that touches O or P and joins the loop again makes the allocator spill inside it.  A reference to move leaves the
        // loop, takes a slow step if that was in the middle of a stage, and comes back.
        acc_t sc[RT][2];
        u32x4_t pc[RT];
#pragma unroll
        for (int x = 0; x < RT; x++) pc[x] = u32x4_t{0, 0, 0, 0};
        slow_step(-1, sc, pc);
        set_references();
        int i = 0;  // the step in front of us; i = 2 st + 1: in the middle of a stage
        while (st < stages) {
            mfma::pin_scalar(careful);  // (or the compiler makes a loop of its own for either value, and spills in them)
            if (!careful && !(i & 1) && i <= steps) {
                acc_t sn[RT][2];     // scores of the odd steps, those of the even ones in sc
                u32x4_t pn[RT];      // P of the even steps, that of the odd ones in pc
                first_fragments(k_of(2 * st + 1));
                bool half = false;
                if ((2 * st + 3) * 32 <= all_open) {
                    do {  // (keys follow that are open to all rows)
                        begin_stage(std::false_type());
                        step(std::false_type(), std::false_type(), 2 * st, sc, sn, pc, pn);
                        if (some_exceed()) { half = true; break; }
                        step(std::false_type(), std::true_type(), 2 * st + 1, sn, sc, pn, pc);
                        st++;
                    } while (!some_exceed() && (2 * st + 3) * 32 <= all_open);
                } else {
                    do {
                        begin_stage(std::true_type());
                        step(std::true_type(), std::false_type(), 2 * st, sc, sn, pc, pn);
                        if (some_exceed()) { half = true; break; }
                        step(std::true_type(), std::true_type(), 2 * st + 1, sn, sc, pn, pc);
                        st++;
                    } while (!some_exceed() && 2 * st <= steps && st < stages);
                }
                i = 2 * st + (half ? 1 : 0);
                if (half) {
#pragma unroll
                    for (int x = 0; x < RT; x++) {
                        sc[x][0] = sn[x][0];
                        sc[x][1] = sn[x][1];
                        pc[x] = pn[x];
                    }
                }
            } else {
                if (!(i & 1)) begin_stage(std::true_type());
                if (i <= steps) slow_step(i, sc, pc);
                if constexpr (PAGED)
                    if (i & 1)
#pragma unroll
                        for (int p = 0; p < G::NI; p++) look_up(st + 4, p);
                i++;
                if (!(i & 1)) st++;
            }
            if (i <= steps && (careful ? some_exceed_scores() : some_exceed())) move_references(pc);
        }
        if (steps == 2 * stages) times_v(steps - 1, pc);  // P V of the last step
    }

    if constexpr (PAGED) {
        if (splits > 1) {
            // A range leaves (reference, sum) and O of its rows, 16 bytes of each lane side by side; the tile's last one to arrive adds
            // them in the order of the ranges.
            constexpr unsigned WAVE = RT * (DT + 1) * 1024, SLICE = 4 * WAVE;
            const __amdgpu_buffer_rsrc_t buf = agent_buffer(ws, ws_bytes);
            const unsigned tile_at = blockIdx.x * gridDim.y * SLICE + wave * WAVE + lane * 16, mine = tile_at + blockIdx.y * SLICE;
            if (wrow0 < rows) {
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    store16_agent(buf, mine + x * (DT + 1) * 1024, f32x4_t{careful ? e_ref[x] : 0.f, careful ? LIFT : e_ref[x], o[x][DT][0], 0.f});
#pragma unroll
                    for (int j = 0; j < DT; j++)
                        store16_agent(buf, mine + (x * (DT + 1) + 1 + j) * 1024, f32x4_t{o[x][j][0], o[x][j][1], o[x][j][2], o[x][j][3]});
                }
            }
            if (!arrive_and_check_last(arrival + blockIdx.x, splits, reinterpret_cast<int *>(smem), tid)) return;
            if (wrow0 < rows) {
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    const unsigned row_at = tile_at + x * (DT + 1) * 1024;
                    // a range's p are 2^(c (s - score) - e): in the common scale its weight is 2^(c score + e)
                    float score = 0.f, e = 0.f, l = 0.f;
                    f32x4_t y[DT];
#pragma unroll
                    for (int j = 0; j < DT; j++) y[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
                    // (four ranges' loads in flight at once)
                    for (int i0 = 0; i0 < splits; i0 += 4) {
                        f32x4_t h[4], part[4][DT];
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const unsigned at = row_at + (i0 + u < splits ? i0 + u : splits - 1) * SLICE;
                            h[u] = load16_agent<f32x4_t>(buf, at);
#pragma unroll
                            for (int j = 0; j < DT; j++) part[u][j] = load16_agent<f32x4_t>(buf, at + (1 + j) * 1024);
                        }
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            if (i0 + u >= splits) break;
                            // the larger of the two stays as it is; one without a key, whose sum is zero, has no say in the scale
                            const float more = __builtin_fmaf(h[u].x - score, c, h[u].y - e);
                            const bool none = h[u].z == 0.f, takes = !none && (l == 0.f || more > 0.f);
                            const float keep = takes ? l == 0.f ? 0.f : __builtin_amdgcn_exp2f(-more) : 1.f;
                            const float w = none ? 0.f : takes ? 1.f : __builtin_amdgcn_exp2f(more);
                            score = takes ? h[u].x : score;
                            e = takes ? h[u].y : e;
                            l = l * keep + h[u].z * w;
#pragma unroll
                            for (int j = 0; j < DT; j++)
#pragma unroll
                                for (int n2 = 0; n2 < 4; n2++) y[j][n2] = y[j][n2] * keep + part[u][j][n2] * w;
                        }
                    }
                    o[x][DT][0] = l;
#pragma unroll
                    for (int j = 0; j < DT; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[x][j][e] = y[j][e];
                }
            }
            arrival_reset(arrival + blockIdx.x, tid);
        }
    }

    // ---- O / l, one rounding: lane (r, g) holds row r of each tile, head-dim columns 16 j + 4 g + e ----
    int l_end = lane;
    mfma::pin_vector(l_end);  // (the rows are counted anew: kept from the beginning they take a register that the loops want)
    const int r_end = l_end & 15, g_end = l_end >> 4;
#pragma unroll
    for (int x = 0; x < RT; x++) {
        const int row = wrow0 + 16 * x + r_end;
        const float l = o[x][DT][0];
        const float inv = l == 0.f ? 0.f : (F8 ? a.v_scale[kvh] : 1.f) / l;  // a row without keys is zero
        if (row >= rows) continue;
        const int tok = quot(row, a.by_group), head = kvh * a.group + row - tok * a.group;
        uint16_t *dst = O + ((long)(q0 + tok) * a.heads + head) * D;
#pragma unroll
        for (int j = 0; j < DT; j++)
            *reinterpret_cast<u32x2_t *>(dst + 16 * j + 4 * g_end) =
                u32x2_t{pack2<CK>(o[x][j][0] * inv, o[x][j][1] * inv), pack2<CK>(o[x][j][2] * inv, o[x][j][3] * inv)};
    }
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
    // rows of a sequence and key / value head, on average
    const long sequences = g.q_tokens < g.batch ? g.q_tokens : g.batch, avg_rows = g.q_tokens * a.group / sequences;
    const long cus = ctx->props.multiProcessorCount;
    // A launch of wide tiles, with the keys of a tile in `splits` ranges
    auto launch = [&](auto kernel, int rows, int d, int splits, int lds, const char *name) -> int {
        const long blocks = (sequences + g.q_tokens * a.group / rows) * g.kv_heads;
        if (blocks > 0x7FFFFFFFL) return HODU_ROCM_UNSUPPORTED;
        if (blocks > kArrivalSlots) splits = 1;
        const size_t ws_bytes = splits > 1 ? (size_t)blocks * splits * rows * (d + 16) * 4 : 0;
        if (splits > 1) {
            if (int rc = ensure_workspace(ctx, ws_bytes)) return rc;
            if (int rc = ensure_arrival(ctx)) return rc;
        }
        if (int rc = ensure_dynamic_lds(ctx, reinterpret_cast<const void *>(kernel), lds)) return rc;
        ctx->last_kernel = name;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks, (unsigned)splits), dim3(W_NT), lds, ctx->stream, qp, kp, vp, (uint16_t *)out, a,
                           (float *)ctx->workspace.ptr, (unsigned)ws_bytes, ctx->arrival);
        return HODU_ROCM_OK;
    };
    // What a launch of wide tiles takes, in ns: a compute unit works on one at a time, so whole rounds of (what a workgroup costs however
    // short it is, what meeting adds, its stages).  Few tiles over a long cache fill the rounds by cutting the keys; the workspace
    // bounds that at four workgroups per compute unit.  Over 4096 cached tokens, head dim 128, whole keys against cut ones: one
    // chunk of 64 tokens 101 and 31 us, of 256 107 and 40, of 512 112 and 63, of 1024 (a workgroup per unit already: not cut) 127 and 118;
    // 128 rows against 192: one chunk of 64 31 and 40 us, four of 512 209 and 222, 64 prompts of 128 102 and 86, one of 4096 185 and 180.
    const long keys = g.paged ? (long)a.width * a.page.d : g.k_tokens / sequences, max_stages = (keys + W_BK - 1) / W_BK;
    struct Wide { int rows, splits; long ns; };
    auto wide = [&](int rows, long stage_ns) {
        const long tiles = sequences * ((avg_rows + rows - 1) / rows) * g.kv_heads;
        Wide best{rows, 1, 0};
        for (int s = 1; s <= 16; s++) {
            if (s > 1 && (!g.paged || s * W_MIN_STAGES > max_stages || s * tiles > 4 * cus)) break;
            const long ns = (tiles * s + cus - 1) / cus * (11000 + (s > 1 ? 5000 + s * 500 : 0) + max_stages * stage_ns / s);
            if (s == 1 || ns < best.ns) best.splits = s, best.ns = ns;
        }
        return best;
    };
    auto by_form = [&](auto ck, auto d, auto paged, auto f8_) -> int {
        constexpr int CK = decltype(ck)::value, D = decltype(d)::value;
        constexpr bool PAGED = decltype(paged)::value, F8 = decltype(f8_)::value;
        // the wide kernels address the keys of a stage, or those of a page, by 32-bit offsets (64-bit ones cost them 7 %, the
        // kernel for 16 rows nothing: it takes what lies further apart)
        const bool near = PAGED ? a.kc.page < (1L << 32) && a.vc.page < (1L << 32) && a.kc.token < (1L << 32) / a.page.d && a.vc.token < (1L << 32) / a.page.d
                                : a.kc.token < (1L << 25) && a.vc.token < (1L << 25);
        const int pin = ctx->force_tile;  // testing hook: 50 tiles of 16 rows, 51 of 128, 52 of 192 or 256
        constexpr int BIG = 64 * W_TILES<D>;
        const Wide small = wide(128, D == 128 ? 1400 : 950), big = wide(BIG, D == 128 ? 1750 : 1450);
        // from three tiles of 16 rows on (over 4096 cached tokens, head dim 128, 16 rows against 128: 4 requests of 8 tokens (32 rows) 34.5
        // and 31.9 us, of 16 41.5 and 32.1; 16 of 8 59.3 and 59.0, of 16 99 and 60; 64 prompts of 8 tokens 16.8 and 20.1, of 12 23.7 and 20.8)
        const bool wide_rows = avg_rows > 2 * R16;
        if (near && (pin == 52 || (pin < 50 && wide_rows && big.ns < small.ns)))
            return launch(seq_attention_wide_kernel<CK, D, PAGED, F8, W_TILES<D>>, BIG, D, big.splits, WGeom<D, F8, PAGED>::LDS,
                          !PAGED ? "attention_varlen_wide" : F8 ? "attention_paged_wide_f8" : "attention_paged_wide");
        if (near && (pin == 51 || (pin < 50 && wide_rows)))
            return launch(seq_attention_wide_kernel<CK, D, PAGED, F8, 2>, 128, D, small.splits, WGeom<D, F8, PAGED>::LDS,
                          !PAGED ? "attention_varlen_wide128" : F8 ? "attention_paged_wide128_f8" : "attention_paged_wide128");
        // Few tiles over long contexts: the keys are cut across workgroups, to about four per compute unit (64 sequences of up to 8192
        // tokens: 254 us with two and with four, 270 with six, 286 with eight: a workgroup costs some 5 us however short it is).
        // How many of them a tile uses goes by its keys, on the device.
        typedef R16Geom<D, F8> G;
        const long tiles = (sequences + g.q_tokens * a.group / R16) * g.kv_heads;
        const long most_keys = PAGED ? (long)a.width * a.page.d : g.k_tokens;
        long splits = 4 * cus / tiles;
        const long worth = (most_keys / R16_BK + R16_MIN_BLOCKS) / R16_MIN_BLOCKS;
        splits = splits > worth ? worth : splits;
        splits = splits > 64 ? 64 : splits;
        if (splits < 1 || tiles > kArrivalSlots) splits = 1;
        const size_t ws_bytes = splits > 1 ? (size_t)tiles * splits * R16 * G::LINE * 4 : 0;
        if (splits > 1) {
            if (int rc = ensure_workspace(ctx, ws_bytes)) return rc;
            if (int rc = ensure_arrival(ctx)) return rc;
        }
        const auto kernel = seq_attention_r16_kernel<CK, D, PAGED, F8>;
        if (tiles > 0x7FFFFFFFL) return HODU_ROCM_UNSUPPORTED;
        if (int rc = ensure_dynamic_lds(ctx, reinterpret_cast<const void *>(kernel), G::LDS)) return rc;
        ctx->last_kernel = !PAGED ? "attention_varlen_r16" : F8 ? "attention_paged_r16_f8" : "attention_paged_r16";
        hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)splits), dim3(R16_NT), G::LDS, ctx->stream, qp, kp, vp, (uint16_t *)out, a,
                           (float *)ctx->workspace.ptr, (unsigned)ws_bytes, ctx->arrival);
        return HODU_ROCM_OK;
    };
    auto by_type = [&](auto ck, auto d) -> int {
        if (!g.paged) return by_form(ck, d, std::false_type(), std::false_type());
        return f8 ? by_form(ck, d, std::true_type(), std::true_type()) : by_form(ck, d, std::true_type(), std::false_type());
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
