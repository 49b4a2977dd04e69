#!/bin/bash
# Builds libtst_hip.so (gfx950) next to the Python package. No fast-math, no fp contraction: the kernels
# rely on a fixed fp32 operation order.  A translation unit that fails to compile fails the build: its stale
# object is removed first, and every compile job's status is checked.
set -e
cd "$(dirname "$0")"
OUT=../libtst_hip.so
# No packed fp32 instructions: some of their forms have given wrong results on this hardware now and then (the host pass does not
# know the feature and says so: harmless).
FLAGS="--offload-arch=gfx950 -O3 -fPIC -ffp-contract=off -std=c++17 -Wall -Wno-unused-result -Xclang -target-feature -Xclang -packed-fp32-ops"
UNITS="capi gemm_f32 gemm_f32_wreg gemm_f32_dma chain_f32 gemm_bf16 gru_fused rowops attn attn_mfma select gumbel paged cache4 prompt rules step"
# One compile job; its kernels may not spill vector registers (check_spills.py says why).
compile() {
  /opt/rocm/bin/hipcc $FLAGS $2 -Rpass-analysis=kernel-resource-usage -c $1.hip -o $1.o.new 2> $1.o.log || { cat $1.o.log >&2; return 1; }
  grep -A3 "warning:" $1.o.log >&2 || true
  python3 check_spills.py $1 < $1.o.log || return 1
  mv $1.o.new $1.o
}
pids=()
for f in $UNITS; do
  if [ ! -f $f.o ] || [ $f.hip -nt $f.o ] || [ build.sh -nt $f.o ] || [ check_spills.py -nt $f.o ] || [ tst_common.h -nt $f.o ] || [ ../../include/tst_hip.h -nt $f.o ]; then
    rm -f $f.o
    EXTRA=""
    # the attention kernels do vector arithmetic on matrix accumulators all the time: keep those in ordinary registers
    case $f in cache4|prompt) EXTRA="-mllvm -amdgpu-mfma-vgpr-form=1" ;; esac
    compile $f "$EXTRA" &
    pids+=($!)
  fi
done
for p in "${pids[@]}"; do
  wait "$p" || { echo "build.sh: a compile job failed" >&2; exit 1; }
done
OBJS=""
for f in $UNITS; do OBJS="$OBJS $f.o"; done
/opt/rocm/bin/hipcc --offload-arch=gfx950 -shared -fPIC -o $OUT $OBJS
# the checked calls of the prompted-decoding kernels, a host-only extension module
# (its fields are torch's: another torch or Python wants another build)
CALLS=../_tst_calls.so
FOR=$(python3 -c "import importlib.metadata as m, sys; print(m.version('torch'), sys.version)")
if [ ! -f $CALLS ] || [ calls.cpp -nt $CALLS ] || [ build.sh -nt $CALLS ] || [ ../../include/tst_hip.h -nt $CALLS ] || [ "$(cat calls.o.for 2> /dev/null)" != "$FOR" ]; then
  rm -f $CALLS
  TORCH=$(python3 -c "import importlib.util as u; print(u.find_spec('torch').submodule_search_locations[0])")
  PY=$(python3 -c "import sysconfig; print(sysconfig.get_path('include'))")
  g++ -O2 -std=c++17 -fPIC -shared -fvisibility=hidden -Wall -D_GLIBCXX_USE_CXX11_ABI=1 -I../../include -I$PY -I$TORCH/include \
    -I$TORCH/include/torch/csrc/api/include calls.cpp -o $CALLS -L$TORCH/lib -ltorch_python -ltorch_cpu -lc10
  echo "$FOR" > calls.o.for
fi
echo "built $OUT"
