// The two bookkeeping operators around attention over a paged cache of keys and values: block tables and slot maps from
// request lengths, and new keys and values into their slots.
#include "common.hpp"
#include "device_types.hpp"

namespace hodu {
namespace {

// ---- block tables and slot maps -----------------------------------------------------------------------------------
// held_r = ceil(cached_r / P), need_r = ceil((cached_r + added_r) / P); a request's fresh pages are the next
// need_r - held_r of the free list, its tokens the next added_r rows: both are running sums over the requests.  The
// sums are over a few hundred requests at most times, the slots over the tokens (a prompt batch: 700 thousand, 4 bytes each):
// every workgroup makes the sums for itself in LDS and then takes its share of the slots, so that nothing has to pass
// between workgroups and one launch does it.  A token's page is computed from the sums (an entry that was in the table before, or the free
// list's), never read back from what another workgroup may be writing.
constexpr int PLAN_NT = 256;
constexpr int PLAN_MAX_BATCH = 16384;  // 8 bytes of LDS each

struct DevPlan {
    int batch, width, n_free, capacity;
    FixedDiv page;
};

// inclusive running sum over the workgroup's threads of v, carried on from `carry`; all threads call
__device__ __forceinline__ long running_sum(long v, long &carry, long *ws) {
    const int tid = threadIdx.x;
    ws[tid] = v;
    __syncthreads();
    for (int step = 1; step < PLAN_NT; step *= 2) {
        const long add = tid >= step ? ws[tid - step] : 0;
        __syncthreads();
        ws[tid] += add;
        __syncthreads();
    }
    const long mine = carry + ws[tid], all = ws[PLAN_NT - 1];
    __syncthreads();
    carry += all;
    return mine;
}

__global__ __launch_bounds__(PLAN_NT) void paged_plan_kernel(const int *__restrict__ cached, const int *__restrict__ added,
                                                             const int *__restrict__ free_pages, int *table, int *__restrict__ lens,
                                                             int *__restrict__ offsets, int *__restrict__ slots, int *__restrict__ used,
                                                             DevPlan p) {
    HODU_DYNAMIC_LDS(smem);
    int *at = reinterpret_cast<int *>(smem);       // [batch + 1]: offsets
    int *first = at + p.batch + 1;                 // [batch]: a request's first page on the free list
    long *ws = reinterpret_cast<long *>(smem + (((long)p.batch * 2 + 1) * 4 + 15) / 16 * 16);  // [PLAN_NT]
    const int tid = threadIdx.x;
    const long row_tokens = (long)p.width * p.page.d;
    long pages = 0, tokens = 0, taken = 0, dealt = 0, refused = 0;
    for (int base = 0; base < p.batch; base += PLAN_NT) {
        const int r = base + tid;
        const int c = r < p.batch ? cached[r] : 0, n = r < p.batch ? added[r] : 0;
        const bool fits = c >= 0 && n >= 0 && (long)c + n <= row_tokens;
        const int held = fits ? fixed_quotient(c, p.page) + (fixed_quotient(c, p.page) * (long)p.page.d < c) : 0;
        const int end = fits ? c + n : 0;
        const int need = fits ? fixed_quotient(end, p.page) + (fixed_quotient(end, p.page) * (long)p.page.d < end) : 0;
        const int fresh = need - held;
        const long to = running_sum(fresh, pages, ws);
        const bool paged = fits && (fresh == 0 || to <= p.n_free);
        const int asked = paged ? n : 0;
        const long row = running_sum(asked, tokens, ws);
        // (the ones that pass the capacity are the last ones with any token: the running sums of those before them are
        // the true offsets, and theirs is where the last accepted one ended)
        const bool ok = paged && (asked == 0 || row <= p.capacity);
        const long true_end = running_sum(ok ? asked : 0, dealt, ws);
        (void)running_sum(ok ? fresh : 0, taken, ws);
        (void)running_sum(r < p.batch && !ok ? 1 : 0, refused, ws);
        if (r < p.batch) {
            at[r] = (int)(true_end - (ok ? asked : 0));
            first[r] = ok ? (int)(to - fresh) : -1;
            if (blockIdx.x == 0) {
                lens[r] = ok ? end : c > 0 ? c : 0;
                offsets[r] = at[r];
            }
        }
    }
    if (tid == 0) at[p.batch] = (int)dealt;
    if (blockIdx.x == 0 && tid == 0) {
        offsets[p.batch] = (int)dealt;
        used[0] = (int)taken;
        used[1] = (int)refused;
    }
    __syncthreads();
    // fresh pages into the tables: a wavefront per request
    const int waves = gridDim.x * (PLAN_NT / 64), wave = blockIdx.x * (PLAN_NT / 64) + (tid >> 6);
    for (int r = wave; r < p.batch; r += waves) {
        if (first[r] < 0) continue;
        const int c = cached[r], end = c + (at[r + 1] - at[r]);
        const int held = (int)(((long)c + p.page.d - 1) / p.page.d), need = (int)(((long)end + p.page.d - 1) / p.page.d);
        for (int i = tid & 63; i < need - held; i += 64) table[(long)r * p.width + held + i] = free_pages[first[r] + i];
    }
    // slots
    const int total = at[p.batch];
    for (long t = (long)blockIdx.x * PLAN_NT + tid; t < p.capacity; t += (long)gridDim.x * PLAN_NT) {
        int slot = -1;
        if (t < total) {
            int lo = 0, hi = p.batch - 1;  // the last request that begins at or before t and has a token there
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (at[mid] <= t) lo = mid; else hi = mid - 1;
            }
            const int c = cached[lo], pos = c + (int)(t - at[lo]);
            const int held = (int)(((long)c + p.page.d - 1) / p.page.d), col = fixed_quotient(pos, p.page);
            const int page = col < held ? table[(long)lo * p.width + col] : free_pages[first[lo] + col - held];
            slot = page * p.page.d + (pos - col * p.page.d);
        }
        slots[t] = slot;
    }
}

// ---- new keys and values into their slots ----------------------------------------------------------------------------
// One copy: a thread moves 8 elements of a head (16 bytes read; 16 or, as 8-bit floats, 8 written) of k and of v.  Bound by memory.
struct DevStore {
    int tokens, heads, per_head;  // per_head: groups of 8 elements
    int n_slots;
    long k_token, k_head, v_token, v_head;
    PagedSide kc, vc;
    FixedDiv page, by_token, by_head;  // by_token: groups of a token, by_head: groups of a head
};

template <bool F8, bool F16>
__device__ __forceinline__ void store8(void *dst, long at, const u32x4_t &x, float scale) {
    if constexpr (!F8) {
        *reinterpret_cast<u32x4_t *>(static_cast<uint16_t *>(dst) + at) = x;
    } else {
        float f[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = x[i];
            f[2 * i] = (F16 ? f16_bits_to_f32((uint16_t)w) : bf16_bits_to_f32((uint16_t)w)) / scale;
            f[2 * i + 1] = (F16 ? f16_bits_to_f32((uint16_t)(w >> 16)) : bf16_bits_to_f32((uint16_t)(w >> 16))) / scale;
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
        const int t = (int)(i / p.by_token.d), rest = (int)(i - (long)t * p.by_token.d);
        const int h = fixed_quotient(rest, p.by_head), e = (rest - h * p.by_head.d) * 8;
        const int slot = slots[t];
        if (slot < 0 || slot >= p.n_slots) continue;
        const int page = fixed_quotient(slot, p.page), in = slot - page * p.page.d;
        const u32x4_t kx = *reinterpret_cast<const u32x4_t *>(k + t * p.k_token + h * p.k_head + e);
        const u32x4_t vx = *reinterpret_cast<const u32x4_t *>(v + t * p.v_token + h * p.v_head + e);
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
    p.page = fixed_div((int)a.page_size);
    const int lds = (int)((a.batch * 2 + 1) * 4 + 15) / 16 * 16 + PLAN_NT * 8;
    if (int rc = ensure_dynamic_lds(ctx, reinterpret_cast<const void *>(paged_plan_kernel), 160 * 1024)) return rc;
    ctx->last_kernel = "paged_plan";
    // a workgroup per 2048 slots, as long as that leaves the sums each of them repeats the smaller part
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
    p.tokens = (int)a.tokens; p.heads = (int)a.kv_heads; p.per_head = (int)(a.d / 8);
    p.n_slots = (int)(a.n_pages * a.page_size);
    p.k_token = a.k_token; p.k_head = a.k_head; p.v_token = a.v_token; p.v_head = a.v_head;
    p.kc = a.kc; p.vc = a.vc;
    p.page = fixed_div((int)a.page_size);
    p.by_token = fixed_div((int)(a.kv_heads * (a.d / 8)));
    p.by_head = fixed_div(p.per_head);
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
