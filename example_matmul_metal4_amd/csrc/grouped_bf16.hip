// Products grouped by expert, bf16 (mtk_grouped_bf16_*).
#define MTK_GROUPED_DT mtk::DT_BF16
#define MTK_GROUPED_NAME(x) mtk_grouped_bf16_##x
#include "grouped_kernels.hpp"
