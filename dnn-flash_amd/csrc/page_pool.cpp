// Host bookkeeping of a paged key-value cache: which sequence holds which
// pages, how many hold each, and what has to be copied when that changes.

#include "onednn_flash_hip.h"

#include <algorithm>
#include <cstring>
#include <functional>
#include <limits>
#include <map>
#include <mutex>
#include <string>
#include <vector>

#include "capi_shared.h"

using ofh::api_error;

struct ofh_page_pool {
    struct Sequence {
        size_t length = 0;
        std::vector<int32_t> pages;
    };
    std::mutex mu;
    size_t num_pages = 0, page_size = 0;
    std::vector<uint32_t> holders;  // sequences that hold a page
    std::vector<int32_t> free;      // min-heap of the pages that none holds; capacity num_pages
    std::map<int64_t, Sequence> sequences;
    int64_t next = 0;

    size_t pages_of(size_t length) const { return (length + page_size - 1) / page_size; }
    int32_t take() {  // (there is one)
        std::pop_heap(free.begin(), free.end(), std::greater<int32_t>());
        const int32_t p = free.back();
        free.pop_back();
        holders[(size_t)p] = 1;
        return p;
    }
    void drop(int32_t p) {
        if (--holders[(size_t)p] != 0) return;
        free.push_back(p);
        std::push_heap(free.begin(), free.end(), std::greater<int32_t>());
    }
};

namespace {

int unknown(int64_t sequence) {
    return api_error(OFH_ERROR_INVALID_ARGUMENT, "unknown sequence " + std::to_string(sequence));
}

// (Where not even the message finds memory, the last one stays.)
int out_of_memory() {
    try {
        return api_error(OFH_ERROR_HIP, "page pool: out of host memory");
    } catch (...) {
        return OFH_ERROR_HIP;
    }
}

// Runs `body` under the pool's lock; no exception leaves the C ABI.
template <typename F>
int guarded(ofh_page_pool* pool, F&& body) {
    if (pool == nullptr) return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool must be non-null");
    try {
        std::lock_guard<std::mutex> lock(pool->mu);
        return body();
    } catch (...) {
        return out_of_memory();
    }
}

}  // namespace

extern "C" {

int ofh_page_pool_create(size_t num_pages, size_t page_size, ofh_page_pool** pool) {
    if (pool == nullptr) return api_error(OFH_ERROR_INVALID_ARGUMENT, "pool must be non-null");
    *pool = nullptr;
    if (num_pages == 0 || num_pages > (size_t)std::numeric_limits<int32_t>::max())
        return api_error(OFH_ERROR_INVALID_ARGUMENT, "num_pages must be positive and fit 31 bits");
    if (page_size == 0 || page_size > ((size_t)1 << 30))
        return api_error(OFH_ERROR_INVALID_ARGUMENT, "page_size must be positive and at most 2^30");
    ofh_page_pool* p = nullptr;
    try {
        p = new ofh_page_pool;
        p->num_pages = num_pages;
        p->page_size = page_size;
        p->holders.assign(num_pages, 0);
        p->free.resize(num_pages);
        for (size_t i = 0; i < num_pages; ++i) p->free[i] = (int32_t)i;  // ascending: a min-heap
    } catch (...) {
        delete p;
        return out_of_memory();
    }
    *pool = p;
    return OFH_SUCCESS;
}

int ofh_page_pool_destroy(ofh_page_pool* pool) {
    delete pool;
    return OFH_SUCCESS;
}

int ofh_page_pool_add(ofh_page_pool* pool, int64_t* sequence) {
    if (sequence == nullptr) return api_error(OFH_ERROR_INVALID_ARGUMENT, "sequence must be non-null");
    return guarded(pool, [&] {
        pool->sequences.emplace(pool->next, ofh_page_pool::Sequence{});
        *sequence = pool->next++;
        return (int)OFH_SUCCESS;
    });
}

int ofh_page_pool_extend(ofh_page_pool* pool, const int64_t* sequences, const size_t* tokens, size_t count,
                         int32_t* copy_src, int32_t* copy_dst, size_t* copies) {
    if (copies == nullptr || (count > 0 && (sequences == nullptr || tokens == nullptr || copy_src == nullptr ||
                                            copy_dst == nullptr)))
        return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool extend: pointers must be non-null");
    *copies = 0;
    return guarded(pool, [&]() -> int {
        // first what it takes, then all of it
        std::vector<ofh_page_pool::Sequence*> seqs(count);
        std::vector<int64_t> order(sequences, sequences + count);
        std::sort(order.begin(), order.end());
        if (std::adjacent_find(order.begin(), order.end()) != order.end())
            return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool extend: a sequence is given twice");
        std::map<int32_t, uint32_t> replaced;  // shared last pages: holders that leave
        size_t need = 0;
        for (size_t i = 0; i < count; ++i) {
            auto it = pool->sequences.find(sequences[i]);
            if (it == pool->sequences.end()) return unknown(sequences[i]);
            ofh_page_pool::Sequence& s = it->second;
            seqs[i] = &s;
            if (tokens[i] > ((size_t)1 << 30) || s.length + tokens[i] > ((size_t)1 << 30))
                return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool extend: a sequence holds at most 2^30 tokens");
            if (tokens[i] == 0) continue;
            const size_t more = pool->pages_of(s.length + tokens[i]) - s.pages.size();
            need += more;
            s.pages.reserve(s.pages.size() + more);
            if (s.length % pool->page_size != 0) {
                const int32_t last = s.pages.back();
                if (pool->holders[(size_t)last] > 1 + replaced[last]) {  // the last holder left keeps the page
                    ++replaced[last];
                    ++need;
                }
            }
        }
        if (need > pool->free.size())
            return api_error(OFH_ERROR_OUT_OF_PAGES, "page pool extend: needs " + std::to_string(need) +
                                                         " pages, " + std::to_string(pool->free.size()) + " are free");
        size_t n = 0;
        for (size_t i = 0; i < count; ++i) {
            ofh_page_pool::Sequence& s = *seqs[i];
            if (tokens[i] == 0) continue;
            if (s.length % pool->page_size != 0 && pool->holders[(size_t)s.pages.back()] > 1) {
                copy_src[n] = s.pages.back();
                copy_dst[n] = pool->take();
                --pool->holders[(size_t)copy_src[n]];
                s.pages.back() = copy_dst[n++];
            }
            s.length += tokens[i];
            while (s.pages.size() < pool->pages_of(s.length)) s.pages.push_back(pool->take());
        }
        *copies = n;
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_fork(ofh_page_pool* pool, int64_t sequence, int64_t* child) {
    if (child == nullptr) return api_error(OFH_ERROR_INVALID_ARGUMENT, "child must be non-null");
    return guarded(pool, [&]() -> int {
        auto it = pool->sequences.find(sequence);
        if (it == pool->sequences.end()) return unknown(sequence);
        const auto made = pool->sequences.emplace(pool->next, it->second).first;
        for (int32_t p : made->second.pages) ++pool->holders[(size_t)p];
        *child = pool->next++;
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_truncate(ofh_page_pool* pool, int64_t sequence, size_t length) {
    return guarded(pool, [&]() -> int {
        auto it = pool->sequences.find(sequence);
        if (it == pool->sequences.end()) return unknown(sequence);
        ofh_page_pool::Sequence& s = it->second;
        if (length > s.length)
            return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool truncate: the sequence has fewer tokens");
        s.length = length;
        while (s.pages.size() > pool->pages_of(length)) {
            pool->drop(s.pages.back());
            s.pages.pop_back();
        }
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_free(ofh_page_pool* pool, int64_t sequence) {
    return guarded(pool, [&]() -> int {
        auto it = pool->sequences.find(sequence);
        if (it == pool->sequences.end()) return unknown(sequence);
        for (int32_t p : it->second.pages) pool->drop(p);
        pool->sequences.erase(it);
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_compact(ofh_page_pool* pool, int32_t* copy_src, int32_t* copy_dst, size_t capacity,
                          size_t* copies) {
    if (copies == nullptr || (capacity > 0 && (copy_src == nullptr || copy_dst == nullptr)))
        return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool compact: pointers must be non-null");
    *copies = 0;
    return guarded(pool, [&]() -> int {
        // the highest used pages at or past the number in use go to the lowest free ones below it
        const size_t used = pool->num_pages - pool->free.size();
        std::vector<int32_t> to(pool->num_pages, -1);
        size_t n = 0, dst = 0;
        for (size_t src = pool->num_pages; src-- > used && n < capacity;) {
            if (pool->holders[src] == 0) continue;
            while (pool->holders[dst] != 0) ++dst;
            to[src] = (int32_t)dst;
            copy_src[n] = (int32_t)src;
            copy_dst[n++] = (int32_t)dst++;
        }
        for (size_t i = 0; i < n; ++i)
            std::swap(pool->holders[(size_t)copy_src[i]], pool->holders[(size_t)copy_dst[i]]);
        for (auto& kv : pool->sequences)
            for (int32_t& p : kv.second.pages)
                if (to[(size_t)p] >= 0) p = to[(size_t)p];
        pool->free.clear();  // (its capacity stays)
        for (size_t p = 0; p < pool->num_pages; ++p)
            if (pool->holders[p] == 0) pool->free.push_back((int32_t)p);
        *copies = n;
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_table(ofh_page_pool* pool, const int64_t* sequences, size_t count, int32_t* table,
                        size_t max_pages, int32_t* lengths) {
    if (count > 0 && (sequences == nullptr || table == nullptr || lengths == nullptr))
        return api_error(OFH_ERROR_INVALID_ARGUMENT, "page pool table: pointers must be non-null");
    return guarded(pool, [&]() -> int {
        for (size_t i = 0; i < count; ++i) {
            auto it = pool->sequences.find(sequences[i]);
            if (it == pool->sequences.end()) return unknown(sequences[i]);
            if (it->second.pages.size() > max_pages)
                return api_error(OFH_ERROR_INVALID_ARGUMENT,
                                 "page pool table: sequence " + std::to_string(sequences[i]) + " holds " +
                                     std::to_string(it->second.pages.size()) + " pages, a row " +
                                     std::to_string(max_pages));
        }
        for (size_t i = 0; i < count; ++i) {
            const ofh_page_pool::Sequence& s = pool->sequences.find(sequences[i])->second;
            int32_t* row = table + i * max_pages;
            std::copy(s.pages.begin(), s.pages.end(), row);
            std::fill(row + s.pages.size(), row + max_pages, -1);
            lengths[i] = (int32_t)s.length;
        }
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_length(ofh_page_pool* pool, int64_t sequence, size_t* length) {
    if (length == nullptr) return api_error(OFH_ERROR_INVALID_ARGUMENT, "length must be non-null");
    return guarded(pool, [&]() -> int {
        auto it = pool->sequences.find(sequence);
        if (it == pool->sequences.end()) return unknown(sequence);
        *length = it->second.length;
        return OFH_SUCCESS;
    });
}

int ofh_page_pool_info(ofh_page_pool* pool, size_t* pages_in_use, size_t* sequences) {
    return guarded(pool, [&] {
        if (pages_in_use != nullptr) *pages_in_use = pool->num_pages - pool->free.size();
        if (sequences != nullptr) *sequences = pool->sequences.size();
        return (int)OFH_SUCCESS;
    });
}

}  // extern "C"
