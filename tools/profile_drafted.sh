# Profile set behind profiles/drafted_*.csv (run from the repo root): times of the drafted-decoding operators and of a drafted decode, kernel
# durations, bytes at the memory, and the counters of the wide trees and the chains (counter passes of their own, few calls each).
set -e
cd /tmp && export TMPDIR=/tmp
R=$GRAFT_REPO_ROOT
O=$R/gpurun_out/drafted
mkdir -p $O/keep
cd $R
timeout -k 10 120 python3 -u tools/drafted_times.py $O/keep/drafted_times.csv
timeout -k 10 200 python3 -u tools/drafted_probe.py $O/keep/drafted_decode.csv
timeout -s KILL 120 rocprofv3 --kernel-trace -d $O/t -o t --output-format csv -- python3 tools/drafted_times.py --trace > $O/keep/trace.log 2>&1
python3 tools/drafted_times.py --summary $(find $O/t -name "*kernel_trace.csv") $O/keep/drafted_kernel_times.csv
rm -rf $O/t
pmc() {  # pmc <tag> <text> <counters...>
  tag=$1 text=$2; shift 2
  timeout -s KILL 120 rocprofv3 --pmc "$@" -d $O/$tag -o p --output-format csv -- python3 tools/drafted_times.py --calls 3 "$text" > $O/keep/$tag.log 2>&1
  echo "pmc $tag done"
}
pmc f "" FETCH_SIZE
pmc w "" WRITE_SIZE
pmc s1 "attend" SQ_BUSY_CU_CYCLES SQ_WAVE_CYCLES SQ_VALU_MFMA_BUSY_CYCLES SQ_ACTIVE_INST_VALU SQ_LDS_IDX_ACTIVE SQ_LDS_BANK_CONFLICT SQ_WAIT_INST_ANY GRBM_GUI_ACTIVE
pmc s2 "attend" SQ_ACTIVE_INST_ANY SQ_ACTIVE_INST_LDS SQ_INSTS_LDS SQ_INSTS_MFMA SQ_INSTS_SALU SQ_INSTS_VALU SQ_WAIT_ANY GRBM_GUI_ACTIVE
python3 tools/pmc_summary.py $O/keep/bytes_all.csv $O/f $O/w
python3 tools/pmc_summary.py $O/keep/attend_all.csv $O/s1 $O/s2
head -1 $O/keep/bytes_all.csv > $O/keep/drafted_hbm_bytes.csv
grep -E "tree_attn|tree_join|paged_|accept_" $O/keep/bytes_all.csv >> $O/keep/drafted_hbm_bytes.csv
head -1 $O/keep/attend_all.csv > $O/keep/drafted_attend_counters.csv
grep -E "tree_attn|tree_join" $O/keep/attend_all.csv >> $O/keep/drafted_attend_counters.csv
rm -rf $O/f $O/w $O/s1 $O/s2 $O/keep/*_all.csv
ls $O/keep
