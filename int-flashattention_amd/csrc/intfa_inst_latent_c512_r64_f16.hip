#include "intfa_latent_attn.h"
namespace intfa { INTFA_DECL_LATENT(launch_latent_c512_r64_f16) { return launch_latent<512, 64, 0>(p, rows, stream); } }
