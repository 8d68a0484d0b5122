// The two bookkeeping operators around attention over a paged cache of keys and values: block tables and slot maps from
// request lengths, and new keys and values into their slots.
#include "common.hpp"
#include "device_types.hpp"

namespace hodu {
namespace {

// ---- block tables and slot maps -----------------------------------------------------------------------------------
// held_r = ceil(cached_r / P), need_r = ceil((cached_r + added_r) / P); a request's fresh pages are the next
// need_r - held_r of the free list, its tokens the next added_r rows: both are running sums over the requests.  There are a few
// hundred requests at most times and up to a million slots (4 bytes each, which is what it has to write): every workgroup makes the
// sums for itself in LDS and then takes its share of the slots, so that nothing has to pass between workgroups and one launch
// does it.  A token's page comes from the sums (an entry that was in the table before, or the free list's), never from what
// another workgroup may be writing.  Bound by latency: two trips to memory and a few barriers, then the slots: 8 requests of a token
// each 5.3 us (of which a launch that does nothing is 1.8), 512 prompts of 700 000 tokens in all 8.2 us.  Running sums by halving
// strides through LDS, a barrier each, took 19 us for the latter: a wavefront sums by itself, four sums meet at one barrier.
//
// The sums saturate at 2^32 - 1 (a saturating sum of non-negative numbers does not depend on its order), which is beyond any
// list or capacity; who is refused is refused in order, so that what was dealt out is where the first refused request stood.
constexpr int PLAN_NT = 256;
constexpr int PLAN_MAX_BATCH = 8192;  // 12 bytes of LDS each

struct DevPlan {
    int batch, width, n_free, capacity;
    int most_pages;  // that 32-bit slots number
    FixedDiv page;
    int wide;  // slots are 16-byte aligned
};

__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }
// inclusive running sum over the wavefront's lanes: shifts by 1, 2, 4, 8 within rows of 16 lanes, each row's last lane to the
// next row, lane 31 to the upper half
__device__ __forceinline__ unsigned running_sum64(unsigned v) {
    v = add_sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, true));
    v = add_sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, true));
    v = add_sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, true));
    v = add_sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, true));
    v = add_sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false));
    v = add_sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false));
    return v;
}
// the same over the workgroup, carried on from `carry`, which moves on; ws: 4 words that no other call of the iteration uses
__device__ __forceinline__ unsigned running_sum(unsigned v, unsigned &carry, unsigned *ws) {
    const int wave = threadIdx.x >> 6;
    unsigned sum = running_sum64(v);
    if ((threadIdx.x & 63) == 63) ws[wave] = sum;
    __syncthreads();
    unsigned before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < PLAN_NT / 64; w++) {
        if (w < wave) before = add_sat(before, ws[w]);
        all = add_sat(all, ws[w]);
    }
    carry = all;
    return add_sat(before, sum);
}

__global__ __launch_bounds__(PLAN_NT) void paged_plan_kernel(const int *__restrict__ cached, const int *__restrict__ added,
                                                             const int *__restrict__ free_pages, int *table, int *__restrict__ lens,
                                                             int *__restrict__ offsets, int *__restrict__ slots, int *__restrict__ used,
                                                             DevPlan p) {
    HODU_DYNAMIC_LDS(smem);
    unsigned *ws = reinterpret_cast<unsigned *>(smem);  // 4 x 4 words for the sums, then:
    int *at = reinterpret_cast<int *>(smem) + 20;       // [batch + 1]: offsets
    int *first = at + p.batch + 1;                      // [batch]: a request's first page on the free list, -1: refused
    int *had = first + p.batch;                         // [batch]: tokens cached
    const int tid = threadIdx.x, wave = tid >> 6;
    const long row_tokens = (long)p.width * p.page.d;
    unsigned pages = 0, tokens = 0, refused = 0, dealt = 0xFFFFFFFFu, taken = 0xFFFFFFFFu;  // the last two: up to the first refused
    for (int base = 0; base < p.batch; base += PLAN_NT) {
        const int r = base + tid;
        const int c = r < p.batch ? cached[r] : 0, n = r < p.batch ? added[r] : 0;
        const bool fits = c >= 0 && n >= 0 && (long)c + n <= row_tokens;
        const int end = fits ? c + n : 0, begin = fits ? c : 0;
        auto pages_of = [&](int t) { const int q = fixed_quotient(t, p.page); return q + (q * p.page.d < t ? 1 : 0); };
        const unsigned fresh = (unsigned)(pages_of(end) - pages_of(begin));
        const unsigned to = running_sum(fresh, pages, ws);
        const bool paged = fits && (fresh == 0 || to <= (unsigned)p.n_free);
        const unsigned asked = paged ? (unsigned)n : 0u;
        const unsigned row = running_sum(asked, tokens, ws + 4);
        const bool ok = paged && (asked == 0 || row <= (unsigned)p.capacity);
        // the wavefront's first refused requests: where the tokens and the list ended, and how many there are
        const unsigned long long no_room = __builtin_amdgcn_ballot_w64(paged && !ok), no_page = __builtin_amdgcn_ballot_w64(fits && !ok && fresh != 0);
        const unsigned long long out = __builtin_amdgcn_ballot_w64(r < p.batch && !ok);
        const unsigned row0 = no_room ? (unsigned)__builtin_amdgcn_readlane((int)(row - asked), (int)__builtin_ctzll(no_room)) : 0xFFFFFFFFu;
        const unsigned to0 = no_page ? (unsigned)__builtin_amdgcn_readlane((int)(to - fresh), (int)__builtin_ctzll(no_page)) : 0xFFFFFFFFu;
        if ((tid & 63) == 0) {
            ws[8 + wave] = row0;
            ws[12 + wave] = to0;
            ws[16 + wave] = (unsigned)__builtin_popcountll(out);
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < PLAN_NT / 64; w++) {
            dealt = ws[8 + w] < dealt ? ws[8 + w] : dealt;
            taken = ws[12 + w] < taken ? ws[12 + w] : taken;
            refused += ws[16 + w];
        }
        if (r < p.batch) {
            const unsigned start = row - asked;
            at[r] = (int)(start < dealt ? start : dealt);
            first[r] = ok ? (fresh ? (int)(to - fresh) : 0) : -1;
            had[r] = c;
            if (blockIdx.x == 0) {
                lens[r] = ok ? end : c > 0 ? c : 0;
                offsets[r] = at[r];
            }
        }
        __syncthreads();
    }
    const int total = (int)(tokens < dealt ? tokens : dealt);
    if (tid == 0) at[p.batch] = total;
    if (blockIdx.x == 0 && tid == 0) {
        offsets[p.batch] = total;
        used[0] = (int)(pages < taken ? pages : taken);
        used[1] = (int)refused;
    }
    __syncthreads();
    // fresh pages into the tables: a wavefront per request
    const int waves = gridDim.x * (PLAN_NT / 64);
    for (int r = blockIdx.x * (PLAN_NT / 64) + wave; r < p.batch; r += waves) {
        if (first[r] < 0) continue;
        const int c = had[r], end = c + (at[r + 1] - at[r]);
        const int held = (int)(((long)c + p.page.d - 1) / p.page.d), need = (int)(((long)end + p.page.d - 1) / p.page.d);
        for (int i = tid & 63; i < need - held; i += 64) table[(long)r * p.width + held + i] = free_pages[first[r] + i];
    }
    // slots, four to a thread
    const long groups = ((long)p.capacity + 3) / 4;
    for (long i = (long)blockIdx.x * PLAN_NT + tid; i < groups; i += (long)gridDim.x * PLAN_NT) {
        const long t0 = 4 * i;
        int slot[4] = {-1, -1, -1, -1};
        if (t0 < total) {
            int lo = 0, hi = p.batch - 1;  // the last request that begins at or before t0 (and so has a token there, or is empty)
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (at[mid] <= t0) lo = mid; else hi = mid - 1;
            }
            int col = -1, first_slot = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int t = (int)t0 + k;
                if (t >= total) break;
                while (t >= at[lo + 1]) lo++, col = -1;
                const int pos = had[lo] + (t - at[lo]), q = fixed_quotient(pos, p.page);
                if (q != col) {
                    const int held = fixed_quotient(had[lo], p.page) + (fixed_quotient(had[lo], p.page) * p.page.d < had[lo] ? 1 : 0);
                    const int page = q < held ? table[(long)lo * p.width + q] : free_pages[first[lo] + q - held];
                    // (a page that is none, or whose slots 32 bits do not hold, gives no slot: wrapped around it would be another token's)
                    first_slot = (unsigned)page < (unsigned)p.most_pages ? page * p.page.d : -1;
                    col = q;
                }
                slot[k] = first_slot < 0 ? -1 : first_slot + (pos - q * p.page.d);
            }
        }
        if (p.wide && t0 + 4 <= p.capacity) {
            *reinterpret_cast<i32x4_t *>(slots + t0) = i32x4_t{slot[0], slot[1], slot[2], slot[3]};
        } else {
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (t0 + k < p.capacity) slots[t0 + k] = slot[k];
        }
    }
}

// ---- new keys and values into their slots ----------------------------------------------------------------------------
// One copy: a thread moves 8 elements of a head (16 bytes read; 16 or, as 8-bit floats, 8 written) of k and of v.  Bound by memory.
// cache[slot] = k or k / scale: 16 bytes of k and of v per thread and turn, neighbouring threads on neighbouring bytes of a head.
// Bound by memory: 16384 tokens of 8 heads of 128 out of a joint projection into an 8-bit cache, 101 MB, 20 us under the profiler, 5.0 TB/s (a
// copy of 1 GB: 5.1).  A full division for each element took 23.6 us, the division of an index by a 64-bit one among it.
struct DevStore {
    int tokens, n_slots;
    long k_token, k_head, v_token, v_head;
    PagedSide kc, vc;
    FixedDiv page, by_token, by_head;  // by_token: groups of 8 elements of a token, by_head: of a head
};

// x / s rounded to nearest, r = 1 / s rounded to nearest: one correction of x r by its exact remainder gives the quotient as the
// division does (P. Markstein, 1990), in three instructions instead of some ten.  Infinite results stay as they are; scales
// outside 2^-100 .. 2^100, where the remainder or r could leave the normal range, are divided by.
__device__ __forceinline__ float quotient(float x, float s, float r, bool plain) {
    if (plain) return x / s;
    const float q = x * r, fixed = __builtin_fmaf(__builtin_fmaf(-q, s, x), r, q);
    return __builtin_fabsf(q) == INFINITY ? q : fixed;
}

template <bool F8, bool F16>
__device__ __forceinline__ void store8(void *dst, long at, const u32x4_t &x, float scale) {
    if constexpr (!F8) {
        *reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(dst) + at) = x;
    } else {
        const float r = 1.0f / scale;
        const bool plain = !(scale > 0x1p-100f && scale < 0x1p100f);
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = x[i];
            f[2 * i] = quotient(F16 ? f16_bits_to_f32((uint16_t)w) : bf16_bits_to_f32((uint16_t)w), scale, r, plain);
            f[2 * i + 1] = quotient(F16 ? f16_bits_to_f32((uint16_t)(w >> 16)) : bf16_bits_to_f32((uint16_t)(w >> 16)), scale, r, plain);
        }
        *reinterpret_cast<u32x2_t *>(static_cast<uint8_t *>(dst) + at) =
            u32x2_t{f32x4_to_f8e4m3_sat(f[0], f[1], f[2], f[3]), f32x4_to_f8e4m3_sat(f[4], f[5], f[6], f[7])};
    }
}

template <bool F8, bool F16>
__global__ __launch_bounds__(256) void paged_store_kernel(const uint16_t *__restrict__ k, const uint16_t *__restrict__ v,
                                                          void *__restrict__ k_cache, void *__restrict__ v_cache,
                                                          const int *__restrict__ slots, const float *__restrict__ k_scale,
                                                          const float *__restrict__ v_scale, DevStore p) {
    const long groups = (long)p.tokens * p.by_token.d, step = (long)gridDim.x * 256;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < groups; i += step) {
        const int t = groups <= 0x7FFFFFFF ? fixed_quotient((int)i, p.by_token) : (int)(i / p.by_token.d);
        const int rest = (int)(i - (long)t * p.by_token.d), h = fixed_quotient(rest, p.by_head), e = (rest - h * p.by_head.d) * 8;
        const int slot = slots[t];
        const u32x4_t kx = *reinterpret_cast<const u32x4_t *>(k + t * p.k_token + h * p.k_head + e);
        const u32x4_t vx = *reinterpret_cast<const u32x4_t *>(v + t * p.v_token + h * p.v_head + e);
        if (slot < 0 || slot >= p.n_slots) continue;
        const int page = fixed_quotient(slot, p.page), in = slot - page * p.page.d;
        store8<F8, F16>(k_cache, page * p.kc.page + in * p.kc.token + h * p.kc.head + e, kx, F8 ? k_scale[h] : 1.f);
        store8<F8, F16>(v_cache, page * p.vc.page + in * p.vc.token + h * p.vc.head + e, vx, F8 ? v_scale[h] : 1.f);
    }
}

}  // namespace

int launch_paged_plan(hodu_rocm_ctx *ctx, const int *cached, const int *added, const int *free_pages, int *table, int *lens,
                      int *offsets, int *slots, int *used, const PagedPlanArgs &a) {
    if (a.batch > PLAN_MAX_BATCH) return fail(HODU_ROCM_UNSUPPORTED, "paged_plan: at most %d requests, got %ld", PLAN_MAX_BATCH, a.batch);
    DevPlan p{};
    p.batch = (int)a.batch; p.width = (int)a.width; p.n_free = (int)a.n_free; p.capacity = (int)a.capacity;
    p.most_pages = (int)((1L << 31) / a.page_size < 0x7FFFFFFF ? (1L << 31) / a.page_size : 0x7FFFFFFF);
    p.page = fixed_div((int)a.page_size);
    p.wide = (uintptr_t)slots % 16 == 0;
    const int lds = (int)(20 + 3 * a.batch + 1) * 4;
    if (int rc = ensure_dynamic_lds(ctx, reinterpret_cast<const void *>(paged_plan_kernel), 160 * 1024)) return rc;
    ctx->last_kernel = "paged_plan";
    // two groups of four slots to a thread, as long as that leaves the sums that each workgroup repeats the smaller part
    long blocks = (a.capacity + 2047) / 2048;
    blocks = blocks < 1 ? 1 : blocks > 512 ? 512 : blocks;
    hipLaunchKernelGGL(paged_plan_kernel, dim3((unsigned)blocks), dim3(PLAN_NT), lds, ctx->stream, cached, added, free_pages, table, lens,
                       offsets, slots, used, p);
    HODU_HIP(hipGetLastError());
    return HODU_ROCM_OK;
}

int launch_paged_store(hodu_rocm_ctx *ctx, int dtype, int cache_dtype, const void *k, const void *v, void *k_cache, void *v_cache,
                       const int *slots, const float *k_scale, const float *v_scale, const PagedStoreArgs &a) {
    auto al = [](long e) { return e % 8 == 0; };
    for (long e : {a.d, a.k_token, a.k_head, a.k_off, a.v_token, a.v_head, a.v_off, a.kc.page, a.kc.token, a.kc.head, a.kc.off, a.vc.page,
                   a.vc.token, a.vc.head, a.vc.off})
        if (!al(e)) return HODU_ROCM_UNSUPPORTED;
    if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || (uintptr_t)k_cache % 16 || (uintptr_t)v_cache % 16) return HODU_ROCM_UNSUPPORTED;
    const bool f8 = cache_dtype == HODU_F8E4M3, f16 = dtype == HODU_F16;
    DevStore p{};
    p.tokens = (int)a.tokens;
    p.n_slots = (int)(a.n_pages * a.page_size);
    p.k_token = a.k_token; p.k_head = a.k_head; p.v_token = a.v_token; p.v_head = a.v_head;
    p.kc = a.kc; p.vc = a.vc;
    p.page = fixed_div((int)a.page_size);
    p.by_token = fixed_div((int)(a.kv_heads * (a.d / 8)));
    p.by_head = fixed_div((int)(a.d / 8));
    const size_t es = f8 ? 1 : 2;
    const uint16_t *ks = (const uint16_t *)k + a.k_off, *vs = (const uint16_t *)v + a.v_off;
    void *kd = (char *)k_cache + a.kc.off * es, *vd = (char *)v_cache + a.vc.off * es;
    const long groups = a.tokens * p.by_token.d;
    long blocks = (groups + 255) / 256;
    if (blocks > 8192) blocks = 8192;
    auto launch = [&](auto kernel, const char *name) {
        ctx->last_kernel = name;
        hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, ctx->stream, ks, vs, kd, vd, slots, k_scale, v_scale, p);
    };
    if (!f8) launch(paged_store_kernel<false, false>, "paged_store");
    else if (f16) launch(paged_store_kernel<true, true>, "paged_store_f16_f8");
    else launch(paged_store_kernel<true, false>, "paged_store_bf16_f8");
    HODU_HIP(hipGetLastError());
    return HODU_ROCM_OK;
}

}  // namespace hodu
