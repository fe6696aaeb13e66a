#include "intfa_paged_decode.h"
namespace intfa { INTFA_DECL_PAGED(launch_paged_d128) { return launch_paged<128>(p, sel, stream); } }
