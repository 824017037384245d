# Phase times inside strip_kernel<Dense> (stats and grad pass): a DIAGNOSTIC copy of the library (-DHCM_STRIP_TIMING:
# s_memtime stamps of wave 0 of every workgroup, summed per phase of the key-tile loop), built here and loaded through HCM_LIB.
# usage (GPU box): strip_timing.sh
R=${GRAFT_REPO_ROOT:-/root/repo}
D=/tmp/stripdiag
rm -rf $D && mkdir -p $D/hcmoco_amd/csrc $D/include && cp $R/include/*.h $D/include/ && cp $R/hcmoco_amd/csrc/*.hip $R/hcmoco_amd/csrc/*.h $R/hcmoco_amd/csrc/Makefile $D/hcmoco_amd/csrc/ && cd $D/hcmoco_amd/csrc
# the product's own rules and flags, with one macro more
make -s -j16 libhcmoco_hip.so HIPCC="/opt/rocm/bin/hipcc -DHCM_STRIP_TIMING" || exit 1
HCM_LIB=$D/hcmoco_amd/csrc/libhcmoco_hip.so python $R/tools/probes/strip_timing.py
