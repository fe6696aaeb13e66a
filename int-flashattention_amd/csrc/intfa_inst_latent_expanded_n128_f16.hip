#include "intfa_latent_expanded.h"
namespace intfa { INTFA_DECL_EXPANDED(launch_expanded_n128_f16) { return launch_expanded<128, 64, 128, 0>(p, causal, stream); } }
