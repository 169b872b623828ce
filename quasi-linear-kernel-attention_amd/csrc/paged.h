// A cache of keys and values in pages and the attention that reads it: what the host side (paged_api.hip) and the
// kernel files share. Not part of the public interface.
#pragma once

#include <hip/hip_runtime.h>
#include <cstddef>
#include <cstdint>

#include "paged_cut.h"
#include "qlka.h"

namespace qlka {

struct PgStrides { uint32_t page, head, row; };                // of pages, in bytes (one instruction a product)
struct PgOut { int64_t b, h, r; };

// How a launch's work is cut (paged_device.h): workgroups aimed at for each key head, the least positions of a part,
// the launch's size, and where the parts' sums go: [unit][rows of a block][padded D], and [unit][rows][2] (reference,
// sum).
struct PgUnits {
    float aim;
    int least, groups;
    int64_t room;                            // units that the workspace has places for
    float *part, *part2;
    int* table;                              // of many sequences (paged_join.hip, paged_table), else null
};

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
    pg::Division page_division;
    float scale, q_sign;                     // |scale|; its sign (or 0)
    PgUnits step, tiles;                     // few rows (paged_step.h), chunks (paged_tiles.h); groups 0: not in a call
    int few;                                 // sequences of more rows a key head are the tiles'
    int blocks;                              // of rows (paged_read)
};

constexpr int BLOCK = 32;                    // elements of a row that share an exponent
constexpr int LEAST_EXP = 27;
constexpr int PG_ALIGN = 128;                // positions of a part: a multiple
constexpr int PG_LOOKED_UP = 320;            // sequences that every workgroup looks up by itself: 64, then the others
constexpr int PG_STEP_ROWS = 16;             // rows (of the heads that share a key head) of the step kernel's blocks
constexpr int PG_READ_ROWS = 2;               // rows of a lane that reads the cache back
constexpr int PG_TILE_ROWS = 128;            // of the tiles' workgroups

// Launchers; each returns a hipError_t value.
int pg_write(int dtype, int held, const PgParams& p, hipStream_t st);
int pg_read(int dtype, int held, const PgParams& p, hipStream_t st);
int pg_attend_bf16(int held, const PgParams& p, hipStream_t st);
int pg_attend_f32(int held, const PgParams& p, hipStream_t st);
int pg_table(const PgParams& p, hipStream_t st);
int pg_join(int dtype, const PgParams& p, hipStream_t st);

}  // namespace qlka
