#include "paged.h"
namespace l3p_pg {
int init_f32(l3p_paged_ctx*) { return L3P_OK; }
int launch_f32(l3p_paged_ctx* ctx, int, const void*, long long, void*, long long, cudaStream_t) { return L3P_E_UNSUPPORTED; }
}
