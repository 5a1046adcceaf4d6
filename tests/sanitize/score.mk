# The same for the calls on scores (score_api.cpp): run as `make -f score.mk _build/score_san`.
include Makefile

SCORE_OBJS = $(LIB)/_build/score_attention.o $(LIB)/_build/score_tiles.o $(LIB)/_build/score_weights.o \
             $(LIB)/_build/score_evict.o

_build/score_host_san.o: $(LIB)/csrc/score_api.cpp $(wildcard $(ROOT)/include/*.h) $(wildcard $(LIB)/csrc/*.hpp) | _build
	$(HIPCC) -x hip --offload-arch=$(ARCH) -O1 -g -std=c++17 -fPIC $(HSAN) \
	  -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-command-line-argument \
	  -I$(ROOT)/include -I$(LIB)/csrc -c $< -o $@

_build/driver_score.o: driver_score.cpp $(wildcard $(ROOT)/include/*.h) | _build
	$(HIPCC) -x c++ -O1 -g -std=c++17 $(HSAN) -Wall -I$(ROOT)/include -c $< -o $@

_build/score_san: _build/api_host_san.o _build/score_host_san.o _build/driver_score.o $(KERNEL_OBJS) $(SCORE_OBJS)
	$(HIPCC) --offload-arch=$(ARCH) $(HSAN) -o $@ _build/driver_score.o _build/score_host_san.o _build/api_host_san.o \
	  $(KERNEL_OBJS) $(SCORE_OBJS) -L/opt/rocm/lib -lrocprofiler-sdk-roctx -Wl,-rpath,/opt/rocm/lib
