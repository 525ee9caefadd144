"""Direct loads into LDS: the wait state between the write of M0 and the load that reads it, in the built assembly."""
import re
import subprocess

from peco_amd import _native

SOURCE = """
#include "common.hpp"
using namespace peco;
__global__ void loads(const uint16_t* src, uint32_t* out, uint32_t off) {
    __shared__ __align__(16) uint32_t tile[3 * 256];
    dma16(src + 8 * threadIdx.x, lds_addr(tile));
    dma16_off(src, 16 * threadIdx.x + off, lds_addr(tile + 256));
    dma4(src + 2 * threadIdx.x, lds_addr(tile + 512));
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    out[threadIdx.x] = tile[threadIdx.x] + tile[256 + threadIdx.x] + tile[512 + threadIdx.x];
}
"""


def test_m0_is_written_a_wait_state_before_the_load(tmp_path):
    source, listing = tmp_path / "loads.hip", tmp_path / "loads.s"
    source.write_text(SOURCE)
    subprocess.run([_native._hipcc(), *_native.HIP_FLAGS, "-I", str(_native.CSRC), "-S", "--offload-device-only",
                    str(source), "-o", str(listing)], check=True, capture_output=True)
    code = [line.split(";")[0].split() for line in listing.read_text().splitlines()]
    code = [words for words in code if words and re.match(r"[a-z]+_", words[0])]
    loads = [i for i, words in enumerate(code) if words[0].startswith("global_load_lds")]
    assert len(loads) == 3
    for i in loads:
        assert "m0," not in code[i - 1], f"{' '.join(code[i - 1])} right before {' '.join(code[i])}"
