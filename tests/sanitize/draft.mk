# The same for the drafted-tree half (draft_api.cpp): run as `make -f draft.mk _build/draft_san`.
include Makefile

DRAFT_OBJS = $(LIB)/_build/draft_attention.o $(LIB)/_build/draft_tiles.o $(LIB)/_build/draft_cache.o

_build/draft_host_san.o: $(LIB)/csrc/draft_api.cpp $(wildcard $(ROOT)/include/*.h) $(wildcard $(LIB)/csrc/*.hpp) | _build
	$(HIPCC) -x hip --offload-arch=$(ARCH) -O1 -g -std=c++17 -fPIC $(HSAN) \
	  -Xclang -target-feature -Xclang -packed-fp32-ops -Wno-unused-command-line-argument \
	  -I$(ROOT)/include -I$(LIB)/csrc -c $< -o $@

_build/driver_draft.o: driver_draft.cpp $(wildcard $(ROOT)/include/*.h) | _build
	$(HIPCC) -x c++ -O1 -g -std=c++17 $(HSAN) -Wall -I$(ROOT)/include -c $< -o $@

_build/draft_san: _build/api_host_san.o _build/draft_host_san.o _build/driver_draft.o $(KERNEL_OBJS) $(DRAFT_OBJS)
	$(HIPCC) --offload-arch=$(ARCH) $(HSAN) -o $@ _build/driver_draft.o _build/draft_host_san.o _build/api_host_san.o \
	  $(KERNEL_OBJS) $(DRAFT_OBJS) -L/opt/rocm/lib -lrocprofiler-sdk-roctx -Wl,-rpath,/opt/rocm/lib
