// k_attend_pages.hip -- attention of a batch's new tokens over a paged KV
// cache (vkml_attend_pages): softmax(q k^T scale) v over each token's keys,
// the ones that a group shares through its first sequence's table, the rest
// through the sequence's own.
#include <hip/hip_runtime.h>

#include <string>

#include "device.hpp"
#include "internal.hpp"
#include "pages.hpp"

using namespace vkml::dev;
using vkml::pages::Batch;

namespace {

struct PagesArgs {
    const float* q;  // [tokens, heads, hd]
    const void* k;
    const void* v;
    const int32_t* table;
    float* out;
    Batch batch;
    uint64_t page_stride;
    uint32_t heads, kv_heads, page_size, pages, table_stride;
    float scale, softcap;
};

// A wave per (head, token), a key at a time: the running maximum m, the sum l
// of e^(x - m) and the sum o of e^(x - m) v.
template <typename T, int HD>
__global__ void __launch_bounds__(64) k_attend_pages(PagesArgs a) {
    constexpr int N = HD / 64;
    const int32_t t = static_cast<int32_t>(blockIdx.x);
    const uint32_t h = blockIdx.y, lane = threadIdx.x, kvh = h / (a.heads / a.kv_heads);
    int32_t s = t;
    if (a.batch.starts) {
        s = 0;
        for (int32_t i = 0; i < a.batch.seqs; i += 64) {
            const int32_t j = i + static_cast<int32_t>(lane);
            s += __popcll(__ballot(j < a.batch.seqs && a.batch.start(j + 1) <= t));
        }
    }
    if (s >= a.batch.seqs || t < a.batch.start(s)) return;
    const int32_t end = a.batch.length(s) - a.batch.count(s) + t - a.batch.start(s) + 1;
    const int32_t g = a.batch.group_of(s), shared = g < 0 ? 0 : a.batch.group_shared(g);
    const int32_t first = g < 0 ? s : a.batch.group_start(g);
    const uint64_t row = (static_cast<uint64_t>(t) * a.heads + h) * HD;
    float q[N], o[N], m = -__FLT_MAX__, l = 0.0f;
    for (int i = 0; i < N; ++i) q[i] = a.q[row + 64 * i + lane], o[i] = 0.0f;
    for (int32_t j = 0; j < max(end, shared); ++j) {
        const int32_t page = a.table[static_cast<uint64_t>(j < shared ? first : s) * a.table_stride + j / a.page_size];
        if (static_cast<uint32_t>(page) >= a.pages) continue;
        const uint64_t at = static_cast<uint64_t>(page) * a.page_stride + (static_cast<uint64_t>(kvh) * a.page_size + j % a.page_size) * HD + lane;
        float x = 0.0f;
        for (int i = 0; i < N; ++i) x += q[i] * static_cast<float>(static_cast<const T*>(a.k)[at + 64 * i]);
        x = wave_sum(x) * a.scale;
        if (a.softcap > 0.0f) x = a.softcap * tanhf(x / a.softcap);
        const float mn = fmaxf(m, x), f = expf(m - mn), p = expf(x - mn);
        l = l * f + p;
        for (int i = 0; i < N; ++i) o[i] = o[i] * f + p * static_cast<float>(static_cast<const T*>(a.v)[at + 64 * i]);
        m = mn;
    }
    for (int i = 0; i < N; ++i) a.out[row + 64 * i + lane] = l == 0.0f ? 0.0f : o[i] / l;
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

extern "C" {

uint64_t vkml_attend_pages_workspace_bytes(const vkml_attend_pages_params*) { return 0; }

int vkml_attend_pages(const vkml_attend_pages_params* p, const float* q, const void* k_pages, const void* v_pages, const int32_t* table,
                      const int32_t* lengths, const int32_t* starts, const int32_t* group_starts, const int32_t* group_keys, void* workspace,
                      float* out) {
    VKML_REQUIRE_INIT();
    VKML_CHECK_ARG(p, "attend_pages: null params");
    if (const char* why = vkml::pages::check(*p)) return vkml::abi::fail(VKML_ERROR_INVALID_ARGUMENT, std::string("attend_pages: ") + why);
    if (p->seqs == 0 || p->tokens == 0) return VKML_OK;
    VKML_CHECK_ARG(starts || p->tokens == p->seqs, "attend_pages: without starts every sequence has one token");
    VKML_CHECK_ARG(q && k_pages && v_pages && table && lengths && workspace && out && (p->groups == 0 || (group_starts && group_keys)),
                   "attend_pages: null buffer");
    VKML_CHECK_ARG(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(workspace) && aligned16(out),
                   "attend_pages: q, the pools, the workspace and out must be 16-byte aligned");
    const Batch batch{lengths, starts, group_starts, group_keys, static_cast<int32_t>(p->seqs), static_cast<int32_t>(p->tokens),
                      static_cast<int32_t>(p->groups), static_cast<int32_t>(p->table_stride * p->page_size)};
    const uint64_t stride = p->page_stride ? p->page_stride : static_cast<uint64_t>(p->kv_heads) * p->page_size * p->head_dim;
    const PagesArgs a{q, k_pages, v_pages, table, out, batch, stride, p->heads, p->kv_heads, p->page_size, p->pages, p->table_stride, p->scale,
                      p->softcap};
    vkml::abi::ProfileScope prof("attend_pages");
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(p->tokens, p->heads), dim3(64), 0, vkml::abi::stream(), a); };
    if (p->kv_type == VKML_F16) p->head_dim == 128 ? go(k_attend_pages<_Float16, 128>) : go(k_attend_pages<_Float16, 64>);
    else p->head_dim == 128 ? go(k_attend_pages<float, 128>) : go(k_attend_pages<float, 64>);
    return vkml::abi::check_launch("attend_pages");
}

}  // extern "C"
