// Copies of whole pages inside paged caches, all layers of all caches in one launch: a fork's own last page, moves of a
// defragmentation. The page lists come from the host (where the cache's bookkeeping is) and travel as launch parameters.
// Bound by memory: a CTA moves 16 KB, every thread with four 16-byte loads in flight. 101 pages of 131 KB in 16 layers of both caches 129 us
// (6.6 TB/s in and out, the measured copy rate), one page of 32 KB in 32 layers 2.2 us.
#include "exl3_common.cuh"
#include "host_common.h"
#include "spans.h"
#include "../../include/ampstein_b200.h"
#include <cstdlib>

namespace amp {

constexpr int CP_CACHES = 32, CP_PAIRS = 256;  // of one launch: its parameters stay below 4 KB
constexpr int CP_THREADS = 256, CP_EACH = 4;
constexpr int CP_CHUNK = CP_THREADS * CP_EACH * 16;

struct CpParams
{
    unsigned char* base[CP_CACHES];
    long layer[CP_CACHES], page[CP_CACHES];    // strides in bytes
    int src[CP_PAIRS], dst[CP_PAIRS];
    int caches, layers, pairs, chunks;
    long page_bytes;
};

__global__ __launch_bounds__(CP_THREADS)
void copy_pages_kernel(const __grid_constant__ CpParams P)
{
    unsigned int u = blockIdx.x;
    const int chunk = u % P.chunks; u /= P.chunks;
    const int pair = u % P.pairs; u /= P.pairs;
    const int layer = u % P.layers, cache = u / P.layers;
    unsigned char* const at = P.base[cache] + layer * P.layer[cache];
    const unsigned char* const from = at + P.src[pair] * P.page[cache];
    unsigned char* const to = at + P.dst[pair] * P.page[cache];
    const long first = (long) chunk * CP_CHUNK + threadIdx.x * 16;
    uint4 x[CP_EACH];
    #pragma unroll
    for (int i = 0; i < CP_EACH; ++i)
        if (first + i * CP_THREADS * 16 < P.page_bytes) x[i] = *reinterpret_cast<const uint4*>(from + first + i * CP_THREADS * 16);
    #pragma unroll
    for (int i = 0; i < CP_EACH; ++i)
        if (first + i * CP_THREADS * 16 < P.page_bytes) *reinterpret_cast<uint4*>(to + first + i * CP_THREADS * 16) = x[i];
}

// The page lists are in order: inside the pool, no destination twice, no page both copied from and copied to
static int cp_check(const int* src, const int* dst, int n, int pages)
{
    unsigned char* seen = (unsigned char*) calloc((size_t) pages, 1);
    if (!seen) return fail(AMP_E_ARG, "copy_pages: out of host memory");
    int rc = 0;
    for (int i = 0; i < n && !rc; ++i)
    {
        if (src[i] < 0 || src[i] >= pages || dst[i] < 0 || dst[i] >= pages) rc = fail(AMP_E_ARG, "copy_pages: copy %d -> %d outside %d pages", src[i], dst[i], pages);
        else if (seen[dst[i]]) rc = fail(AMP_E_ARG, "copy_pages: page %d is written twice", dst[i]);
        else seen[dst[i]] = 1;
    }
    for (int i = 0; i < n && !rc; ++i)
        if (src[i] != dst[i] && seen[src[i]]) rc = fail(AMP_E_ARG, "copy_pages: page %d is both read and written", src[i]);
    free(seen);
    return rc;
}

// Caches must not share memory (one cache twice may be given: the same bytes to the same places). Their extents in order of address: one of a model's
// dozens of caches meets none or the one beside it.
struct CpExtent { uintptr_t from, to; int cache; };

static int cp_overlap(void* const* caches, const long* layer_strides, const long* page_strides, int n, int layers, int pages, long page_bytes)
{
    if (n < 2) return 0;
    auto span = [&](int i) { return Span(caches[i], page_bytes, { { layers, layer_strides[i] }, { pages, page_strides[i] } }); };
    CpExtent* const e = (CpExtent*) malloc((size_t) n * sizeof(CpExtent));
    if (!e) return fail(AMP_E_ARG, "copy_pages: out of host memory");
    for (int i = 0; i < n; ++i) { const Span s = span(i); e[i] = { s.at, s.at + s.extent(0), i }; }
    qsort(e, n, sizeof(CpExtent), [](const void* a, const void* b) {
        const uintptr_t x = ((const CpExtent*) a)->from, y = ((const CpExtent*) b)->from;
        return x < y ? -1 : x > y ? 1 : 0;
    });
    int rc = 0;
    for (int i = 0; i < n && !rc; ++i)
        for (int j = i + 1; j < n && e[j].from < e[i].to && !rc; ++j)
        {
            const Span a = span(e[i].cache), b = span(e[j].cache);
            if (!apart(a, b) && !a.same(b)) rc = fail(AMP_E_ARG, "copy_pages: caches %d and %d overlap", e[i].cache, e[j].cache);
        }
    free(e);
    return rc;
}

}  // namespace amp

using namespace amp;

AMP_API int amp_b200_copy_pages(void* const* caches, const long* layer_strides, const long* page_strides, int n_caches, int layers,
                                int pages, long page_bytes, const int* src, const int* dst, int n, cudaStream_t stream)
{
    AMP_REQUIRE(n >= 0 && n_caches >= 0 && layers >= 0 && pages >= 0 && page_bytes >= 0, "copy_pages: negative size");
    if (n == 0) return 0;
    AMP_REQUIRE(src && dst && (n_caches == 0 || (caches && layer_strides && page_strides)), "copy_pages: null pointer");
    if (int rc = cp_check(src, dst, n, pages)) return rc;
    AMP_REQUIRE(page_bytes % 16 == 0 && page_bytes <= (1l << 32), "copy_pages: pages of %ld bytes (a multiple of 16)", page_bytes);
    for (int i = 0; i < n_caches; ++i)
    {
        const long ls = layer_strides[i], ps = page_strides[i];
        AMP_REQUIRE(caches[i] && (((uintptr_t) caches[i] | (uintptr_t) ls | (uintptr_t) ps) & 15) == 0, "copy_pages: cache %d: null or not 16-byte aligned", i);
        AMP_REQUIRE((pages == 1 || ps >= page_bytes) && (layers <= 1 || ls >= (pages - 1) * ps + page_bytes || (ls >= page_bytes && (pages == 1 || ps >= (layers - 1) * ls + page_bytes))),
                    "copy_pages: cache %d: its pages overlap", i);
    }
    if (n_caches == 0 || layers == 0 || page_bytes == 0) return 0;
    if (int rc = cp_overlap(caches, layer_strides, page_strides, n_caches, layers, pages, page_bytes)) return rc;
    const long chunks = (page_bytes + CP_CHUNK - 1) / CP_CHUNK;
    CpParams P;
    for (int c0 = 0; c0 < n_caches; c0 += CP_CACHES)
    {
        P.caches = n_caches - c0 < CP_CACHES ? n_caches - c0 : CP_CACHES;
        for (int i = 0; i < P.caches; ++i) { P.base[i] = (unsigned char*) caches[c0 + i]; P.layer[i] = layer_strides[c0 + i]; P.page[i] = page_strides[c0 + i]; }
        for (int at = 0; at < n; )
        {
            int m = 0;
            for (; at < n && m < CP_PAIRS; ++at)
                if (src[at] != dst[at]) { P.src[m] = src[at]; P.dst[m] = dst[at]; ++m; }
            if (m == 0) break;
            P.layers = layers; P.pairs = m; P.chunks = (int) chunks; P.page_bytes = page_bytes;
            const long grid = chunks * m * layers * P.caches;
            AMP_REQUIRE(grid < (1l << 31), "copy_pages: too many bytes in one call");
            copy_pages_kernel<<<(unsigned) grid, CP_THREADS, 0, stream>>>(P);
            if (cudaError_t e = cudaGetLastError()) return cuda_rc(e, "copy_pages launch");
        }
    }
    return 0;
}
