# Phase times inside the row-8 kernels: a DIAGNOSTIC copy of the library (-DHCM_ROW8_TIMING: s_memtime stamps per workgroup),
# built here, loaded by tools/probes/row8_timing.py through HCM_LIB.  usage (on the GPU box): row8_timing.sh [crop] [B]
R=${GRAFT_REPO_ROOT:-/root/repo}
D=/tmp/row8diag
rm -rf $D && mkdir -p $D/hcmoco_amd/csrc $D/include && cp $R/include/*.h $D/include/ && cp $R/hcmoco_amd/csrc/*.hip $R/hcmoco_amd/csrc/*.h $R/hcmoco_amd/csrc/Makefile $D/hcmoco_amd/csrc/ && cd $D/hcmoco_amd/csrc
# the product's own rules and flags, with one macro more
make -s -j16 libhcmoco_hip.so HIPCC="/opt/rocm/bin/hipcc -DHCM_ROW8_TIMING" || exit 1
HCM_LIB=$D/hcmoco_amd/csrc/libhcmoco_hip.so python $R/tools/probes/row8_timing.py ${1:-256} ${2:-32}
