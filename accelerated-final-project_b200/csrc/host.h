// What the entry points outside api.cu share with it: the error message of the calling thread, the launch counter, the
// device's context (SM count, error words) and the library-held workspace.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include <mutex>

#include "../../include/b200attn.h"

namespace b200attn {

int fail(int status, const char *fmt, ...);   // sets b200attn_last_error() and returns `status`
void count_launches(unsigned long long n);
void set_last_path(const char *name);

struct HostCall {
    int dev = 0, sm_count = 0;
    size_t max_smem = 0;             // opt-in shared memory of a CTA, static part included
    unsigned *err_dev = nullptr, *err_sys = nullptr;
    unsigned spin_limit = 0, wait_extra = 0;   // wait_extra: arrivals that a kernel waits for and nobody makes (b200attn_debug_lost_arrival)
    std::unique_lock<std::mutex> lock;   // held by a call that uses the library's workspace, until it has enqueued its work
};
// Looks the current device up; reports what an earlier asynchronous call left behind.
int host_begin(HostCall *c);
// The library's workspace of this device, at least `bytes`: the call is ordered after the device's previous call of that kind.
int host_workspace(HostCall *c, size_t bytes, cudaStream_t st, void **ws);
// Waits for the stream unless the call is asynchronous, and reports kernel errors then.
int host_end(HostCall *c, cudaStream_t st, bool async);

}  // namespace b200attn
