// The routed experts with waits of the tcgen05 kernels that run out within microseconds, as in impatient.cu.
#define CFM_SCREEN_WAIT_NS (blockIdx.x % 8 * 400u)
#define CFM_SCREEN_DRAIN_NS 2000000u
#define CFM_SCREEN_WAIT "test_wait"
#include "cfm_experts.cu"
