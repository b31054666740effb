/*
 * Host build of the rules of g4s_cache.h that the kernels of the 8-bit cache run:
 * division, a row's tokens, places in a plane and scales.
 */
#include "../../gemma4.pas_amd/csrc/g4s_cache.h"

using namespace g4s;

extern "C" {
int32_t t_divide(int32_t n, int32_t d) { return divide(n, divisor(d)); }
/* Divisors `from` to `to` - 1, at the numerators next to their multiples. */
int t_divide_all(int32_t from, int32_t to)
{
    for (int32_t d = from; d < to; ++d) {
        const Divisor v = divisor(d);
        const int64_t most = INT32_MAX / d;
        const int64_t step = most / 97 + 1;
        for (int64_t k = 0;; k = k + step < most ? k + step : most) {
            for (int64_t n = k * d - 1; n <= k * d + 1; ++n)
                if (n >= 0 && n <= INT32_MAX && divide((int32_t)n, v) != n / d) return d;
            if (k == most) break;
        }
        if (divide(INT32_MAX, v) != INT32_MAX / d) return d;
    }
    return 0;
}
void t_row_tokens(const int32_t* starts, const int32_t* lengths, int32_t row, int32_t tokens,
                  int64_t room, int32_t* out)
{
    const RowTokens r = row_tokens(starts, lengths, row, tokens, room);
    out[0] = r.start;
    out[1] = r.count;
    out[2] = r.length;
    out[3] = r.bad;
}
int64_t t_cache_offset(int64_t page_stride, int32_t part_bytes, int32_t token_bytes, int32_t page,
                       int32_t in_page, int32_t head)
{
    CachePool p{};
    p.page_stride = page_stride;
    p.part_bytes = part_bytes;
    p.token_bytes = token_bytes;
    return cache_offset(p, page, in_page, head);
}
int t_scale_ok(uint32_t bits) { return scale_ok(bits); }
int32_t t_scale_exponent(double top) { return scale_exponent(top); }
/* Tiles of a row of `count` tokens from place `from` on that find no slot in the grid
 * of the append (rows one behind the other from token `start` on): 0. */
int32_t t_missing_slots(int32_t start, int32_t count, int32_t from, int32_t tile)
{
    const int32_t starts[2] = {start, start + count};
    const int64_t slots = share_begin(starts, 1, 1, tile, 2) - share_begin(starts, 0, 1, tile, 2);
    const int64_t tiles = count ? (from + count - 1) / tile - from / tile + 1 : 0;
    return (int32_t)(tiles > slots ? tiles - slots : 0);
}
/* The same of blocks of `unit` columns in the grid of the attention. */
int32_t t_missing_blocks(int32_t start, int32_t count, int32_t group, int32_t unit)
{
    const int32_t starts[2] = {start, start + count};
    const int64_t slots =
        share_begin(starts, 1, group, unit, 1) - share_begin(starts, 0, group, unit, 1);
    const int64_t blocks = ((int64_t)count * group + unit - 1) / unit;
    return (int32_t)(blocks > slots ? blocks - slots : 0);
}
/* Whether units are shared out without gaps and unit_group names their workgroup. */
int t_units_shared(int64_t total, int32_t groups)
{
    if (first_unit(total, 0, groups) != 0 || first_unit(total, groups, groups) != total) return 0;
    for (int32_t w = 0; w < groups; ++w) {
        const int64_t a = first_unit(total, w, groups), b = first_unit(total, w + 1, groups);
        if (b <= a || unit_group(a, total, groups) != w || unit_group(b - 1, total, groups) != w)
            return 0;
    }
    return 1;
}
int t_vectors_meet(const int64_t* a, const int64_t* b)
{
    return vectors_meet(Vectors{(uint64_t)a[0], a[1], a[2], a[3], a[4], a[5]},
                        Vectors{(uint64_t)b[0], b[1], b[2], b[3], b[4], b[5]});
}
/* The rows' kernel's share of a call (rows of `counts` tokens, none taken together; those with more columns
 * than kFewCols are the prompts' kernel's): 0, or what is wrong with it.  1: more units than
 * the grid is made for, 2: work is shared among workgroups that the grid does not have, 3: units that are
 * no workgroup's, 4: an item whose parts are not those that its last workgroup waits for. */
int t_rows_share(int32_t head_dim, int32_t kv_heads, int32_t group, int32_t rows, int32_t tokens,
                 const int32_t* counts, int starts, const int32_t* lengths, int64_t room, int32_t window,
                 int32_t ncu)
{
    const RowsShape shape = rows_shape(attend_width(head_dim));
    const int32_t unit = shape.unit(), resident = ncu * (8 / shape.waves);
    const int64_t most = most_units(rows, tokens, starts, kv_heads, group, kFewCols, room, unit);
    const int32_t grid = most < resident ? (int32_t)most : resident;
    int64_t total = 0;
    for (int32_t r = 0; r < rows; ++r) {
        if (is_prompt(counts[r], group, kFewCols)) continue;
        const int32_t first = lengths[r] - counts[r], from = first - window + 1;
        total += (int64_t)column_blocks(counts[r] * group) * kv_heads *
                 place_units(window > 0 && from > 0 ? from : 0, lengths[r], unit);
    }
    if (total > most) return 1;
    const int32_t groups = sharing_groups(total, shape.units, ncu, grid);
    if (groups > grid) return 2;
    if (total == 0) return groups != 0;
    if (first_unit(total, 0, groups) != 0 || first_unit(total, groups, groups) != total) return 3;
    int64_t first = 0;
    for (int32_t r = 0; r < rows; ++r) {
        if (is_prompt(counts[r], group, kFewCols)) continue;
        const int32_t at = lengths[r] - counts[r] - window + 1;
        const int64_t units = place_units(window > 0 && at > 0 ? at : 0, lengths[r], unit);
        for (int32_t i = 0; i < column_blocks(counts[r] * group) * kv_heads; ++i, first += units) {
            const int32_t a = unit_group(first, total, groups);
            const int32_t b = unit_group(first + units - 1, total, groups);
            if (a < 0 || b < a || b >= grid || first_unit(total, a, groups) > first ||
                first_unit(total, b + 1, groups) < first + units)
                return 4;
        }
    }
    return 0;
}
}
