"""Compiles tests/cpp/test_header_layer.cpp against include/anygpu, libanygpu_b200.so and liboracle.so."""
import os
import subprocess

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
OUT = os.path.join(HERE, "_build", "test_header_layer")


def build():
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    src = os.path.join(HERE, "test_header_layer.cpp")
    libdir, orcdir = os.path.join(ROOT, "anygpu_b200", "lib"), os.path.join(ROOT, "oracle")
    cmd = [os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-std=c++17", "-O2", "-x", "cu", "-DAC_WITH_ASSERT",
           "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "include"), src, "-o", OUT,
           "-L", libdir, "-lanygpu_b200", "-L", orcdir, "-loracle",
           "-Xlinker", "-rpath=$ORIGIN/../../../anygpu_b200/lib", "-Xlinker", "-rpath=$ORIGIN/../../../oracle"]
    subprocess.check_call(cmd)
    return OUT


SFT_OUT = os.path.join(HERE, "_build", "sft_dump")


def build_sft_dump():
    """Host-only program around the safetensors reader (compiled with nvcc for the CUDA headers tensor.hpp includes)."""
    os.makedirs(os.path.dirname(SFT_OUT), exist_ok=True)
    cmd = [os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-std=c++17", "-O1", "-x", "cu", "-DAC_WITH_ASSERT",
           "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "include"), os.path.join(HERE, "sft_dump.cpp"),
           "-o", SFT_OUT]
    subprocess.check_call(cmd)
    return SFT_OUT


SCAN_OUT = os.path.join(HERE, "_build", "test_selective_scan_layer")


def build_selective_scan_layer():
    """Compiles tests/cpp/test_selective_scan_layer.cpp against include/anygpu and libanygpu_b200.so."""
    os.makedirs(os.path.dirname(SCAN_OUT), exist_ok=True)
    cmd = [os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-std=c++17", "-O2", "-x", "cu", "-DAC_WITH_ASSERT",
           "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "include"), os.path.join(HERE, "test_selective_scan_layer.cpp"),
           "-o", SCAN_OUT, "-L", os.path.join(ROOT, "anygpu_b200", "lib"), "-lanygpu_b200",
           "-Xlinker", "-rpath=$ORIGIN/../../../anygpu_b200/lib"]
    subprocess.check_call(cmd)
    return SCAN_OUT


LAYOUT_OUT = os.path.join(HERE, "_build", "layout_refusals")
VIEWS_OUT = os.path.join(HERE, "_build", "test_slice_views")


def _build_against_library(out, source, opt):
    os.makedirs(os.path.dirname(out), exist_ok=True)
    cmd = [os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc"), "-std=c++17", opt, "-x", "cu", "-DAC_WITH_ASSERT",
           "-gencode", "arch=compute_100a,code=sm_100a", "-I", os.path.join(ROOT, "include"), os.path.join(HERE, source),
           "-o", out, "-L", os.path.join(ROOT, "anygpu_b200", "lib"), "-lanygpu_b200",
           "-Xlinker", "-rpath=$ORIGIN/../../../anygpu_b200/lib"]
    subprocess.check_call(cmd)
    return out


def build_layout_refusals():
    """Compiles tests/cpp/layout_refusals.cpp against include/anygpu and libanygpu_b200.so (it runs without a GPU)."""
    return _build_against_library(LAYOUT_OUT, "layout_refusals.cpp", "-O0")


def build_slice_views():
    """Compiles tests/cpp/test_slice_views.cpp against include/anygpu and libanygpu_b200.so."""
    return _build_against_library(VIEWS_OUT, "test_slice_views.cpp", "-O1")


if __name__ == "__main__":
    print(build())
    print(build_sft_dump())
    print(build_selective_scan_layer())
    print(build_layout_refusals())
    print(build_slice_views())
