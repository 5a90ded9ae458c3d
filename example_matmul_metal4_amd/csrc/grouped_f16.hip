// Products grouped by expert, f16 (mtk_grouped_f16_*).
#define MTK_GROUPED_DT mtk::DT_F16
#define MTK_GROUPED_NAME(x) mtk_grouped_f16_##x
#include "grouped_kernels.hpp"
