/*
 * Host build of the rules of g4s_pages.h that the page kernels run: a row's
 * step and slots, the geometry's limits and a copy's addresses.
 */
#include "../../gemma4.pas_amd/csrc/g4s_pages.h"

using namespace g4s;

extern "C" {
void t_row_step(int32_t parent, int32_t from_rows, int32_t length, int32_t grow,
                int32_t page_tokens, int32_t max_slots, int64_t* out)
{
    const RowStep s = row_step(parent, from_rows, length, grow, page_tokens, max_slots);
    out[0] = s.length;
    out[1] = s.kept;
    out[2] = s.fresh;
    out[3] = s.tail;
    out[4] = s.bad;
}
int32_t t_used_slots(int64_t tokens, int32_t page_tokens)
{
    return used_slots(tokens, page_tokens);
}
int t_geometry_ok(const g4s_page_geometry* g) { return geometry_ok(*g) ? 1 : 0; }
int64_t t_page_offset(const g4s_page_geometry* g, int32_t plane, int32_t page, uint32_t i,
                      uint32_t per_part, int32_t vec)
{
    return page_offset(*g, plane, page, i, per_part, vec);
}
}
