"""What the host makes of a device's status block, without a GPU: `csrc/api.cu` compiled against a CUDA runtime whose few calls
work on host memory, with reports and split-K arrival counters set by hand."""
import glob
import os
import subprocess

from kaio_b200 import build

HOST = r'''
#include <cuda_runtime.h>
#include <string.h>
static cudaError_t fake_device(int* d) { *d = 0; return cudaSuccess; }
static cudaError_t fake_sync(cudaStream_t) { return cudaSuccess; }
static cudaError_t fake_copy(void* to, const void* from, size_t n, cudaMemcpyKind) { memcpy(to, from, n); return cudaSuccess; }
static cudaError_t fake_set(void* to, int value, size_t n) { memset(to, value, n); return cudaSuccess; }
#define cudaGetDevice fake_device
#define cudaStreamSynchronize fake_sync
#define cudaMemcpy fake_copy
#define cudaMemset fake_set
#include "api.cu"

static uint32_t status[kaio::STATUS_WORDS], counters[5];

// What device_status says: its return value and the code it reports.
static int ask(uint32_t* code)
{
    uint32_t c[4] = {9, 9, 9, 9};
    const int rc = kaio_b200_device_status(nullptr, c);
    *code = c[0];
    return rc;
}

static void report(uint32_t at, uint32_t code, uint32_t site)
{
    const uint32_t words[4] = {code, 7, site, 8};
    memcpy(status + at, words, sizeof words);
}

static bool counters_are(uint32_t value)
{
    for (uint32_t c : counters)
        if (c != value)
            return false;
    return true;
}

int main()
{
    kaio::g_ctx[0].device = 0;
    kaio::g_ctx[0].status = status;
    kaio::StreamScratch scratch;
    scratch.tile_counters = counters;
    scratch.num_tile_counters = 5;
    kaio::g_scratch[0].push_back(&scratch);
    uint32_t code;
    const int rc = check(code);
    kaio::g_scratch[0].clear();
    return rc;
}
'''


def run(tmp_path, check):
    build.build()
    src, exe = tmp_path / "t.cu", tmp_path / "t"
    src.write_text(HOST.replace("int main()", "static int check(uint32_t& code)\n{" + check + "}\n\nint main()"))
    objs = [o for o in glob.glob(os.path.join(build.OBJ_DIR, "*.o")) if os.path.basename(o) != "api.o"]
    r = subprocess.run([build._nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-I", build.CSRC, str(src), *objs,
                        "-o", str(exe), "-cudart", "static", "-ldl"], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, (r.returncode, r.stdout, r.stderr)


def test_a_bad_index_does_not_hide_a_wait_that_gave_up(tmp_path):
    """Both reported, in either order: the timeout comes first and is recovered from, then the index, then nothing."""
    run(tmp_path, r'''
    for (int order = 0; order < 2; ++order) {
        for (uint32_t& c : counters)
            c = 3;
        for (int i = 0; i < 2; ++i) {
            if (i == order)
                report(kaio::STATUS_INDEX, kaio::DEV_BAD_INDEX, 4);
            else
                report(0, kaio::DEV_TIMEOUT, 99);
        }
        if (ask(&code) != KAIO_B200_ERR_TIMEOUT || code != kaio::DEV_TIMEOUT || !counters_are(0))
            return 1;
        if (ask(&code) != KAIO_B200_ERR_INVALID_CONFIG || code != kaio::DEV_BAD_INDEX || !strstr(kaio_b200_last_error(), "q_start"))
            return 2;
        if (ask(&code) != KAIO_B200_OK || code != 0)
            return 3;
    }
    return 0;
''')


def test_a_bad_index_leaves_the_arrival_counters_alone(tmp_path):
    """Nothing gave up: launches on other streams may be counting with them."""
    run(tmp_path, r'''
    for (uint32_t& c : counters)
        c = 3;
    report(kaio::STATUS_INDEX, kaio::DEV_BAD_INDEX, 1);
    if (ask(&code) != KAIO_B200_ERR_INVALID_CONFIG || !counters_are(3))
        return 1;
    if (ask(&code) != KAIO_B200_OK || !counters_are(3))
        return 2;
    report(0, kaio::DEV_TIMEOUT, 99);
    if (ask(&code) != KAIO_B200_ERR_TIMEOUT || !counters_are(0))
        return 3;
    return 0;
''')
