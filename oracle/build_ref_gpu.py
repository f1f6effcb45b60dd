"""Builds oracle/_ref/libferro_ref_gpu.so: ferro's own CUDA kernels for LayerNorm forward and
row softmax, recompiled for sm_100a from the reference sources where they lie, behind a small
launcher (oracle/ref_gpu_launch.cu) that uses the reference's launch geometry.

This is the "reference source recompiled" column of the benchmark: how fast ferro's kernels, as
written, run on the same B200.  It is not ferro as shipped (that needs Rust, cudarc and nvrtc);
it is test / measurement infrastructure, never loaded by the library.

Sources (read in place, nothing is copied into the repository; the generated file and the .so
go to oracle/_ref/, which git ignores):
  crates/ferro-cuda/src/layer_norm.cu            included twice (with and without OUTPUT_ONLY)
  crates/ferro-cuda/src/kernels.rs:536-588       the CUDA text of softmax_row_stats_source() and
                                                 softmax_apply_source(), taken out of the Rust
                                                 raw strings with their format placeholders filled
Usage: python oracle/build_ref_gpu.py [/path/to/ferro]   (default: $FERRO_SOURCE, else where the build
container mounts the reference checkout; when that directory does not exist the script does nothing and
an existing .so is kept).
"""
import os
import re
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
OUT_DIR = os.path.join(HERE, "_ref")
GEN = os.path.join(OUT_DIR, "ref_kernels_generated.cu")
OUT = os.path.join(OUT_DIR, "libferro_ref_gpu.so")
LAUNCHER = os.path.join(HERE, "ref_gpu_launch.cu")


def _raw_string(src, fn_name):
    """The text of the r#"..."# literal inside `pub fn fn_name`."""
    at = src.index(f"pub fn {fn_name}")
    m = re.compile(r'r#"(.*?)"#', re.S).search(src, at)
    return m.group(1)


def _fill(text, **subst):
    for k, v in subst.items():
        text = text.replace("{" + k + "}", str(v))
    return text.replace("{{", "{").replace("}}", "}")


def generate(root):
    rs = open(os.path.join(root, "crates/ferro-cuda/src/kernels.rs")).read()
    block = int(re.search(r"pub const REDUCE_BLOCK: u32 = (\d+);", rs).group(1))
    stats = _fill(_raw_string(rs, "softmax_row_stats_source"), KERNEL_NAME="ref_softmax_row_stats", REDUCE_BLOCK=block)
    apply_src = _raw_string(rs, "softmax_apply_source")
    apply_sm = _fill(apply_src, KERNEL_NAME="ref_softmax_apply", body="expf(x[i] - m) / s")
    apply_log = _fill(apply_src, KERNEL_NAME="ref_log_softmax_apply", body="(x[i] - m) - logf(s)")
    ln = os.path.join(root, "crates/ferro-cuda/src/layer_norm.cu")
    os.makedirs(OUT_DIR, exist_ok=True)
    with open(GEN, "w") as f:
        f.write("// generated by oracle/build_ref_gpu.py from the ferro sources; not part of the repository\n")
        f.write(f"#define REF_REDUCE_BLOCK {block}\n")
        f.write(f'#define ferro_kernel ref_layer_norm\n#include "{ln}"\n#undef ferro_kernel\n')
        f.write(f'#define ferro_kernel ref_layer_norm_output\n#define OUTPUT_ONLY\n#include "{ln}"\n#undef OUTPUT_ONLY\n#undef ferro_kernel\n')
        f.write(stats + apply_sm + apply_log)
    return GEN


DEFAULT_ROOT = os.environ.get("FERRO_SOURCE") or os.path.join(os.sep, "root", "reference")


def build(root=DEFAULT_ROOT, force=False):
    if not os.path.exists(os.path.join(root, "crates", "ferro-cuda", "src", "kernels.rs")):  # an empty folder is no source either
        return OUT if os.path.exists(OUT) else None
    if not force and os.path.exists(OUT) and os.path.getmtime(OUT) >= max(os.path.getmtime(LAUNCHER), os.path.getmtime(__file__)):
        return OUT
    gen = generate(root)
    nvcc = "/usr/local/cuda/bin/nvcc" if os.path.exists("/usr/local/cuda/bin/nvcc") else "nvcc"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-lineinfo", "-shared", "-Xcompiler", "-fPIC",
                    "-include", gen, LAUNCHER, "-o", OUT, "-cudart", "shared"], check=True)
    return OUT


if __name__ == "__main__":
    print(build(sys.argv[1] if len(sys.argv) > 1 else DEFAULT_ROOT, force=True))
