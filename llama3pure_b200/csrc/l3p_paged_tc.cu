#include "paged.h"
namespace l3p_pg {
int tc_tile(const l3p_paged_ctx*) { return 128; }
int tc_rows(const l3p_paged_ctx*) { return 256; }
int init_tc(l3p_paged_ctx*) { return L3P_OK; }
int init_f32(l3p_paged_ctx*) { return L3P_OK; }
int launch_tc(l3p_paged_ctx* ctx, int, const void*, long long, void*, long long, cudaStream_t) { return L3P_E_UNSUPPORTED; }
int launch_f32(l3p_paged_ctx* ctx, int, const void*, long long, void*, long long, cudaStream_t) { return L3P_E_UNSUPPORTED; }
}
