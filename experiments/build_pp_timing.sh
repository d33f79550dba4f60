#!/bin/bash
# Experiment build of the library with -DSDAMD_PP_TIMING (phase timestamps in the ping-pong GEMM kernels, gemm2_kernel.h), by the
# library's own Makefile with its flags: objects under /tmp (or $1), the library at experiments/micro/libsdamd_pptiming.so
# (git-ignored).
set -e
R=$(cd "$(dirname "$0")/.." && pwd)
S=$R/stable-diffusion_amd/csrc
B=${1:-/tmp/pp_timing_build}; mkdir -p $B
make -f $S/Makefile -C $B -j6 --eval "vpath %.hip $S" --eval "vpath %.h $S" EXTRA=-DSDAMD_PP_TIMING
cp $B/libsdamd.so $R/experiments/micro/libsdamd_pptiming.so
ls -la $R/experiments/micro/libsdamd_pptiming.so
