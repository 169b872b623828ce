// A cache of keys and values in pages and the attention that reads it: what the host side (paged_api.hip) and the kernel
// files share. Not part of the public interface.
#pragma once

#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

#include "qlka.h"

namespace qlka {

struct PgStrides { int64_t page, head, row; };                 // of pages, in elements or bytes of exponents
struct PgOut { int64_t b, h, r; };

struct PgParams {
    char *k_pages, *v_pages;
    PgStrides sk, sv;
    uint8_t *k_exp, *v_exp;                  // null unless 8 bits are held
    PgStrides ske, sve;
    const int *tables, *lengths, *offsets;   // offsets null: a token a sequence
    int64_t table_stride;
    const void *q, *k, *v;                   // strides of b are 0
    void *out, *out_k, *out_v;
    PgOut sq, snk, snv, so, sok, sov;
    int B, H, G, T, D, N;
    int page_size, num_pages, table_len;
    int places;                              // positions that a table's row has pages for
    uint32_t magic, shift;                   // n / page_size = n * magic >> shift for n below 2^31
    float scale, q_sign;                     // |scale|; its sign (or 0)
    int splits;                              // of a sequence's keys
    int few;                                 // sequences of more rows a key head are the tiles' (paged_tiles)
    int blocks;                              // of rows: of all sequences (paged_tiles), of each
    int outside;                             // step kernel: it also writes the rows outside every sequence
    float *part, *part2;                     // [split][H][T][padded D], [split][H][T][2], as softmax.h has them
};

constexpr int BLOCK = 32;                    // elements of a row that share an exponent
constexpr int LEAST_EXP = 27;
constexpr int PG_STEP_ROWS = 16;             // rows (of the heads that share a key head) of the step kernel's blocks
constexpr int PG_READ_ROWS = 2;               // rows of a lane that reads the cache back
constexpr int PG_TILE_ROWS = 128;            // of the tiles' workgroups

// Launchers; each returns a hipError_t value.
int pg_write(int dtype, int held, const PgParams& p, hipStream_t st);
int pg_read(int dtype, int held, const PgParams& p, hipStream_t st);
int pg_step(int dtype, int held, const PgParams& p, hipStream_t st);
int pg_tiles(int dtype, int held, const PgParams& p, hipStream_t st);

}  // namespace qlka
