// Launch interface of the paged cache's operators (paged.hip, pages.hip): a plan
// of a step's work, attention over pages with shared prefixes, over selected
// pages, the pages' key bounds and the selection.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llmtie {

// A page is what a slot of the tiled f16 cache is: [kv_heads][blocks of 32
// positions], 2^shift positions. Row t of the table holds the pages of sequence
// t's positions, `cols` of them.
struct Pages {
    const uint16_t* cache;
    const int* table;
    int rows, cols, shift, pages;
};

constexpr int PG_GROUPS = 1024;  // groups of a plan at most
constexpr int PG_COLS = 32;      // (row, query head) columns of a tile at most

// A plan's words: the header, PG_ROW a row, then PG_ITEM an item, the tiles' (the
// wide ones) first.
constexpr int PG_HEAD = 16, PG_ROW = 12, PG_ITEM = 16;
__host__ __device__ constexpr int PG_TILE_ROWS(int group) { return PG_COLS / group; }
// Rows of one sequence that are a tile at least, a quarter of one; and the tiles of such
// rows that an aligned tile of rows can hold, which a plan has room for: four, five of two
// rows where a tile has ten, fewer of fewer rows.
__host__ __device__ constexpr int PG_RUN_ROWS(int group) {
    return PG_TILE_ROWS(group) / 4 > 2 ? PG_TILE_ROWS(group) / 4 : 2;
}
__host__ __device__ constexpr int PG_TILE_RUNS(int group) { return PG_TILE_ROWS(group) / PG_RUN_ROWS(group); }
__host__ __device__ inline size_t plan_items_at(size_t nseq) { return (PG_HEAD + PG_ROW * nseq + 15) / 16 * 16; }
// What an item is: it writes its rows' context, it is of a shared tile.
constexpr int PG_WHOLE = 1, PG_SHARED = 2;
// Parts that a row's context is joined from at most, its own and its group's: the sizes keep to it.
constexpr int PG_PARTS = 1088;
// Pages of a sequence up to which rows that selected pages of it are attended together.
constexpr int PG_UNION = 4096;

struct PagePlanArgs {
    const int* tk;      // [nseq] live positions
    const int* row;     // [nseq] table row, or null: row s
    const int* lo;      // [nseq] first position behind the shared ones, or null
    const int* starts;  // [groups + 1] first rows of the groups, or null
    const int* prefix;  // [groups] leading positions that a group's rows share
    int* plan;
    int nseq, groups, window, shared, rows, cols, shift, group, kv_heads;
    int max_wide, max_own;    // items there is room for
    int target;               // items of a kv head that the work is divided into
    int tile_target;          // and where the most of it is tiles'
    int whole;                // every row is one item (no group shares)
    int together;             // rows of one sequence may follow one another
};
hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t st);

struct PagedArgs {
    Pages p;
    const float* q;  // row r's heads at r * q_stride
    float* out;      // [nseq, heads * hd]
    const int* tk;
    const int* row;      // selected pages only
    const int* chosen;   // selected pages only: [nseq][kv_heads][count]
    const float* slopes;
    const int* plan;     // null: selected pages
    float* part;         // own items' O, then the wide ones', then their (m, l)
    long q_stride;
    int nseq, kv_heads, group;
    int max_wide, max_own;
    int items;           // of a kv head, at most
    int count, runs;     // selected pages: how many, and the workgroups of a (row, kv head)
    int tile_runs;       // and of a tile of rows at most
    int together;        // rows of one sequence may follow one another
    int stream;          // more bytes than are worth keeping in the Infinity Cache
    int merge;           // some row may have partials
    float scale, softcap;
};
hipError_t launch_paged(int hd, const PagedArgs& a, hipStream_t st);

struct PageBoundsArgs {
    Pages p;
    const int* row;  // [nseq], or null: row s
    const int* low;  // [nseq] first new position, or null: 0
    const int* tk;   // [nseq] live positions
    uint16_t* bounds;  // [pages][kv_heads][2][hd]: greatest, least
    int nseq, kv_heads, per;  // pages of a row taken side by side
};
hipError_t launch_page_bounds(int hd, const PageBoundsArgs& a, hipStream_t st);

struct SelectArgs {
    const float* q;
    const uint16_t* bounds;
    const int* table;
    const int* row;
    const int* tk;
    int* chosen;     // [nseq][kv_heads][count]
    double* exact;   // [nseq][kv_heads][wide]
    float* score;    // [nseq][kv_heads][wide], where chunks > 1
    float* worst;    // [nseq][kv_heads][chunks]
    long q_stride;
    int nseq, kv_heads, group, rows, cols, shift, pages, count, first, last;
    int wide;        // pages a row may have (of max_tk), at most cols
    int chunks;      // workgroups that score a (row, kv head)'s pages
};
hipError_t launch_select(int hd, const SelectArgs& a, hipStream_t st);

}  // namespace llmtie
