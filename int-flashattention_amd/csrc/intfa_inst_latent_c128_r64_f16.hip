#include "intfa_latent_attn.h"
namespace intfa { INTFA_DECL_LATENT(launch_latent_c128_r64_f16) { return launch_latent<128, 64, 0>(p, rows, stream); } }
