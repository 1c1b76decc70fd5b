#include "attend_common.cuh"
namespace clover {
bool attend_mma_supported(int, int, int, int) { return false; }
int attend_mma(int, int, int, const AttendArgs*, int, cudaStream_t, int*) { return CLOVER_B200_ERR_UNSUPPORTED; }
}
