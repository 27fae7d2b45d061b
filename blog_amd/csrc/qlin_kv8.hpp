// qlin_kv8.hpp -- the 8-bit attention cache (struct qlin_kv8_cache, qlin_decoder.h) as the kernels see it.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "qlin_decoder.h"

namespace qlin {

constexpr int kKv8Block = QLIN_KV8_BLOCK, kKv8Recent = QLIN_KV8_RECENT;

// Bytes of a block of one key head: key codes, value codes, two scales, 8 bytes that are left alone.
__host__ __device__ constexpr size_t kv8_record_bytes(int head_dim) { return 64 * static_cast<size_t>(head_dim) + 16; }

struct Kv8View {
    uint8_t *pages;
    float *recent;
    const int *table;
    int n_pages, per, kv;  // blocks of a sequence, key heads

    // the page of a sequence's block, -1 if it has none
    __device__ __forceinline__ int page(int seq, int block) const {
        const int64_t at = static_cast<int64_t>(seq) * per + block;
        const int64_t p = table ? table[at] : at;
        return p >= 0 && p < n_pages ? static_cast<int>(p) : -1;
    }
    __device__ __forceinline__ uint8_t *record(int page, int head, size_t bytes) const {
        return pages + (static_cast<size_t>(page) * kv + head) * bytes;
    }
    // keys (j = 0) or values (1) of the last positions, [64][head_dim]
    __device__ __forceinline__ float *ring(int seq, int head, int j, int head_dim) const {
        return recent + (((static_cast<size_t>(seq) * kv + head) * 2 + j) * kKv8Recent) * head_dim;
    }
};

// Bytes of position t's (0 .. 31) codes of the dims d .. d + 3 (d a multiple of 4) in a record: one dword.
__host__ __device__ constexpr int kv8_key_byte(int t, int d) {
    return 1024 * (d / 32) + 256 * (d / 8 % 4) + 16 * (t % 16) + 8 * (t / 16) + d % 8;
}
__host__ __device__ constexpr int kv8_value_byte(int t, int d, int head_dim) {
    const int w = d / 4 + (t % 2) * (head_dim / 4);
    return 32 * head_dim + 1024 * (w / 16) + 256 * (t / 4 % 4) + 16 * (w % 16) + 8 * (t / 16) + 4 * (t / 2 % 2);
}

// The rows of a sequence in a call: positions start .. start + rows - 1, the cache's end after them.
struct Kv8Rows {
    int start, rows, len;
};
__device__ __forceinline__ Kv8Rows kv8_rows(const int *start_pos, const int *n_rows, int seq, int rows, int cap) {
    Kv8Rows r;
    r.rows = n_rows ? min(max(n_rows[seq], 0), rows) : rows;
    // (any int is a start: far ones are brought to where every row is outside, without overflow)
    r.start = min(max(start_pos[seq], -(1 << 30)), cap);
    r.len = min(max(r.start + r.rows, 0), cap);
    return r;
}

}  // namespace qlin
