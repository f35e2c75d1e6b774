// lgx_pages.cpp -- the pages of a paged cache: forking, reserving, copying, freeing
// (kernels in lgx_pages.hip).
#include "lgx_internal.h"

using namespace lgxi;

namespace {

lgx_status check_pool(const lgx_page_pool* pool, const int32_t* page_table, int32_t maxp) {
    if (!pool) return fail(LGX_NULL_POINTER, "pool is NULL");
    if (!pool->ref || !page_table) return fail(LGX_NULL_POINTER, "NULL ref or page_table");
    if (pool->num_pages <= 0 || maxp <= 0 || maxp > 1 << 26)
        return fail(LGX_INVALID_ARGUMENT, "num_pages=%d maxp=%d", pool->num_pages, maxp);
    return LGX_OK;
}

}  // namespace

extern "C" {

lgx_status lgx_pages_fork(lgx_ctx* c, const lgx_page_pool* pool, int32_t* page_table, int32_t* seq_len,
                          const int32_t* src, const int32_t* dst, int32_t S, int32_t n, int32_t maxp, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_pool(pool, page_table, maxp)) != LGX_OK) return st;
        if (!seq_len || !src || !dst) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (S <= 0 || n <= 0 || n > LGX_PAGES_SEQS || maxp > 256 * 65535)
            return fail(LGX_INVALID_ARGUMENT, "%d of %d sequences, maxp %d", n, S, maxp);
        lgx_fork_args a{pool->ref, page_table, seq_len, src, dst, pool->num_pages, S, maxp, n};
        return launch(c, K_PAGES_FORK, dim3((unsigned)n, cdiv(maxp, 256)), dim3(256), a, stream);
    });
}

lgx_status lgx_pages_free(lgx_ctx* c, const lgx_page_pool* pool, int32_t* page_table, const int32_t* keep, int32_t B,
                          int32_t maxp, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_pool(pool, page_table, maxp)) != LGX_OK) return st;
        if (!keep) return fail(LGX_NULL_POINTER, "NULL keep");
        if (B <= 0 || B > 1 << 23 || maxp > 256 * 65535) return fail(LGX_INVALID_ARGUMENT, "B=%d maxp=%d", B, maxp);
        lgx_pages_free_args a{pool->ref, page_table, keep, pool->num_pages, maxp};
        return launch(c, K_PAGES_FREE, dim3((unsigned)B, cdiv(maxp, 256)), dim3(256), a, stream);
    });
}

lgx_status lgx_pages_reserve(lgx_ctx* c, const lgx_page_pool* pool, int32_t* page_table, const int32_t* seq_len,
                             const int32_t* need, int32_t B, int32_t maxp, int32_t* copies, int32_t* n_copies,
                             int32_t* lacking, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if ((st = check_pool(pool, page_table, maxp)) != LGX_OK) return st;
        if (!seq_len || !need || !copies || !n_copies || !lacking) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (B <= 0 || B > LGX_PAGES_SEQS) return fail(LGX_INVALID_ARGUMENT, "B=%d (1..%d)", B, LGX_PAGES_SEQS);
        // needs are summed in 32 bits
        if ((int64_t)B * ((int64_t)maxp + 1) > INT32_MAX)
            return fail(LGX_OUT_OF_BOUNDS, "a table of %d rows of %d entries", B, maxp);
        // a list of the pages found: never more than there are, nor than all entries
        // and one copy per sequence
        const int64_t most = std::min<int64_t>(pool->num_pages, (int64_t)B * ((int64_t)maxp + 1));
        float* ws = nullptr;
        if ((st = ensure_ws(c, (size_t)most * sizeof(int32_t), stream, &ws)) != LGX_OK) return st;
        lgx_reserve_args a{pool->ref, page_table, seq_len, need, copies, n_copies, lacking, (int32_t*)ws,
                           pool->num_pages, B, maxp};
        return launch(c, K_PAGES_RESERVE, dim3(1), dim3(1024), a, stream);
    });
}

lgx_status lgx_pages_copy(lgx_ctx* c, const lgx_page_plane* planes, int32_t n_planes, int32_t num_pages,
                          const int32_t* copies, const int32_t* n_copies, int32_t max_copies, void* stream) {
    return guarded(__func__, [&]() -> lgx_status {
        lgx_status st = enter(c);
        if (st != LGX_OK) return st;
        if (!planes || !copies || !n_copies) return fail(LGX_NULL_POINTER, "NULL tensor pointer");
        if (n_planes <= 0 || num_pages <= 0 || max_copies <= 0 || max_copies > 1 << 23)
            return fail(LGX_INVALID_ARGUMENT, "%d planes, %d pages, %d copies", n_planes, num_pages, max_copies);
        for (int i = 0; i < n_planes; ++i) {
            if (!planes[i].data) return fail(LGX_NULL_POINTER, "plane %d is NULL", i);
            if (planes[i].page_bytes <= 0 || planes[i].page_bytes > INT64_MAX / num_pages)
                return fail(LGX_INVALID_ARGUMENT, "plane %d: %lld bytes per page", i, (long long)planes[i].page_bytes);
        }
        for (int p0 = 0; p0 < n_planes; p0 += LGX_PLANES) {
            const int np = std::min(n_planes - p0, LGX_PLANES);
            lgx_pages_copy_args a{};
            for (int i = 0; i < np; ++i) {
                a.base[i] = (char*)planes[p0 + i].data;
                a.bytes[i] = planes[p0 + i].page_bytes;
            }
            a.copies = copies;
            a.n_copies = n_copies;
            a.max = max_copies;
            a.num_pages = num_pages;
            if ((st = launch(c, K_PAGES_COPY, dim3((unsigned)max_copies, (unsigned)np), dim3(256), a, stream)) != LGX_OK)
                return st;
        }
        return LGX_OK;
    });
}

}  // extern "C"
