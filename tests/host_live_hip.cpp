// The HIP runtime of host_hip.cpp, with the current device the live-cache calls
// ask for and put back.
#include "host_hip.cpp"

static int g_device = 0;
extern "C" {
hipError_t hipGetDevice(int* d) {
    *d = g_device;
    return hipSuccess;
}
}
