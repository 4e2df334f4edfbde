#!/bin/bash
# layer_profile.sh OUT: kernel trace of perf/operators.py's listed cases, then counters of the large ones, each pass a run of its own
out=$1; mkdir -p $out
here=$(cd "$(dirname "$0")" && pwd)
cd /tmp && export TMPDIR=/tmp
timeout -s KILL 120 rocprofv3 --kernel-trace --stats --output-format csv -d $out/trace -o p -- python3 $here/layer_cases.py > $out/trace.log 2>&1 || exit $?
echo "trace done"
pass() { name=$1; shift; timeout -s KILL 90 rocprofv3 --kernel-trace --pmc "$@" --output-format csv -d $out/pmc_$name -o c -- python3 $here/layer_cases.py 786432 64064 65536 > $out/pmc_$name.log 2>&1 || exit $?; echo "pass $name done"; }
pass mfma SQ_WAVES SQ_BUSY_CU_CYCLES SQ_VALU_MFMA_BUSY_CYCLES SQ_ACTIVE_INST_VALU SQ_LDS_BANK_CONFLICT SQ_LDS_IDX_ACTIVE SQ_INSTS_LDS SQ_INSTS_VALU
pass wait SQ_WAVE_CYCLES SQ_WAIT_ANY SQ_WAIT_INST_ANY SQ_WAIT_INST_LDS SQ_ACTIVE_INST_ANY SQ_ACTIVE_INST_VMEM SQ_INSTS_VMEM_RD SQ_INSTS_VMEM_WR GRBM_GUI_ACTIVE
pass fetch FETCH_SIZE
pass write WRITE_SIZE
pass l2 TCC_HIT_sum TCC_MISS_sum TCC_REQ_sum
pass l1 TCP_TCC_READ_REQ_sum TCP_TOTAL_CACHE_ACCESSES_sum TCP_PENDING_STALL_CYCLES_sum TCP_TCC_WRITE_REQ_sum
pass ta TA_BUSY_avr TA_TOTAL_WAVEFRONTS_sum
