// The kernels of paged_attention_rows.cuh for one type of cache (a file of its own: they take a while to compile).
#include "paged_attention_rows.cuh"

namespace lv {

int paged_rows_launch_e4m3(lv_ctx* ctx, const PagedAttn& p, uint32_t rows, uint32_t blocks) { return rows_launch_kind<LV_TYPE_E4M3>(ctx, p, rows, blocks); }

}  // namespace lv
