#include "intfa_paged_prefill.h"
namespace intfa { INTFA_DECL_PAGED(launch_paged_prefill_d128) { return launch_paged_prefill<128>(p, sel, stream); } }
