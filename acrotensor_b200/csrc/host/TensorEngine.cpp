// acro::TensorEngine: parse / bind / plan caches and single or recorded multi-kernel execution.
#include "TensorEngine.hpp"
#include "SliceTensor.hpp"
#include "acro_b200.h"

#include <cuda_runtime.h>
#include <initializer_list>
#include <vector>

namespace acro
{

TensorEngine::TensorEngine() : IsMultiKernelLaunch(false), TheCudaStream(nullptr), ThePeerGroup(nullptr)
{
    SetExecutorType("Cuda");
}

TensorEngine::TensorEngine(const char *bare_exec_type) : IsMultiKernelLaunch(false), TheCudaStream(nullptr), ThePeerGroup(nullptr)
{
    SetExecutorType(bare_exec_type);
}

TensorEngine::TensorEngine(std::string &exec_type) : IsMultiKernelLaunch(false), TheCudaStream(nullptr), ThePeerGroup(nullptr)
{
    SetExecutorType(exec_type);
}

TensorEngine::~TensorEngine() {}

void TensorEngine::SetExecutorType(const char *bare_exec_type)
{
    std::string exec_type(bare_exec_type ? bare_exec_type : "");
    SetExecutorType(exec_type);
}

void TensorEngine::SetExecutorType(std::string &exec_type)
{
    ACROBATIC_ASSERT(exec_type == "Cuda" || exec_type == "CPUInterpreted", "Unknown Executor type:  " + exec_type);
    Clear();
    ExecutorType = exec_type;
}

void TensorEngine::Clear()
{
    ExecutorMap.clear();
    DimensionedKernelMap.clear();
    KernelMap.clear();
    MKLKernels.clear();
    MKLOutputT.clear();
    MKLInputT.clear();
}

void TensorEngine::operator()(const char *bare_kernel_str, Tensor *out, std::vector<Tensor *> &inputs)
{
    std::string kernel_str(bare_kernel_str);
    (*this)(kernel_str, out, inputs);
}

void TensorEngine::Record(std::string &kernel_str, Tensor *output, std::vector<Tensor *> &inputs)
{
    ACROBATIC_ASSERT(output != nullptr && output->IsInitialized(), "Output variable not initilized in:  " + kernel_str);
    for (Tensor *t : inputs)
    {
        ACROBATIC_ASSERT(t != nullptr && t->IsInitialized(), "Input variable not initilized in:  " + kernel_str);
    }
    if (!IsMultiKernelLaunch)
    {
        MKLKernels.clear();
        MKLOutputT.clear();
        MKLInputT.clear();
    }
    TensorKernel *kernel = GetAddTensorKernel(kernel_str);
    DimensionedKernel *bound = GetAddDimensionedKernel(kernel, output, inputs);
    MKLKernels.push_back(bound);
    MKLOutputT.push_back(output);
    MKLInputT.push_back(inputs);
}

void TensorEngine::operator()(std::string &kernel_str, Tensor *output, std::vector<Tensor *> &inputs)
{
    Record(kernel_str, output, inputs);
    if (!IsMultiKernelLaunch)
    {
        KernelExecutor *executor = GetAddKernelExecutor();
        executor->SetCudaStream(TheCudaStream);
        executor->SetPeerGroup(ThePeerGroup);
        executor->ExecuteSingle(output, inputs);
    }
}

std::string TensorEngine::GetImplementation(const char *bare_kernel_str, Tensor *out, std::vector<Tensor *> &inputs)
{
    std::string kernel_str(bare_kernel_str);
    return GetImplementation(kernel_str, out, inputs);
}

std::string TensorEngine::GetImplementation(std::string &kernel_str, Tensor *output, std::vector<Tensor *> &inputs)
{
    ACROBATIC_ASSERT(!IsMultiKernelLaunch, "GetImplementation can't be used inside a multi kernel launch.");
    Record(kernel_str, output, inputs);
    return GetAddKernelExecutor()->GetImplementation();
}

void TensorEngine::BeginMultiKernelLaunch()
{
    ACROBATIC_ASSERT(!IsMultiKernelLaunch, "Trying to BeginMultiKernelLaunch twice.");
    IsMultiKernelLaunch = true;
    MKLKernels.clear();
    MKLOutputT.clear();
    MKLInputT.clear();
}

void TensorEngine::EndMultiKernelLaunch()
{
    ACROBATIC_ASSERT(IsMultiKernelLaunch, "Found an EndMultiKernelLaunch before a BeginMultiKernelLaunch!");
    IsMultiKernelLaunch = false;
    if (MKLKernels.empty()) return;
    KernelExecutor *executor = GetAddKernelExecutor();
    executor->SetCudaStream(TheCudaStream);
    executor->SetPeerGroup(ThePeerGroup);
    executor->ExecuteMulti(MKLOutputT, MKLInputT);
}

std::string TensorEngine::EndMultiKernelLaunchDescribe()
{
    ACROBATIC_ASSERT(IsMultiKernelLaunch, "Found an EndMultiKernelLaunch before a BeginMultiKernelLaunch!");
    IsMultiKernelLaunch = false;
    if (MKLKernels.empty()) return "";
    return GetAddKernelExecutor()->GetImplementation();
}

void TensorEngine::RequireCuda(const char *what)
{
    ACROBATIC_ASSERT(ExecutorType == "Cuda", std::string(what) + ": the CPUInterpreted executor is not part of this library.");
    ACROBATIC_ASSERT(isCudaReady(), std::string(what) + ": No CUDA device is available; this library has no CPU execution path.");
}

void *TensorEngine::Stream() { return TheCudaStream ? TheCudaStream : getCudaStream(); }

namespace
{
void check_abi(int status, const char *what)
{
    if (status != ACRO_B200_OK) throw_error(std::string("acro_b200 ") + what + " failed: " + acro_b200_last_error());
}

// Shape checks shared by the batched matrix operations (kernel/TensorEngine.cpp:627-690).
void check_matrix_batch(Tensor &A, Tensor *Ainv, Tensor *Adet)
{
    const int rank = A.GetRank();
    ACROBATIC_ASSERT(A.IsInitialized(), "Batched matrix operation on an uninitialized tensor.");
    ACROBATIC_ASSERT(rank >= 2, "Can't treat a tensor of rank < 2 as a batch of matrices.");
    ACROBATIC_ASSERT(A.GetDim(rank - 1) == A.GetDim(rank - 2), "Batched matrix operations need square matrices in the last two dims.");
    ACROBATIC_ASSERT(A.GetDim(rank - 1) <= 3, "Batched matrix operations support matrix dims <= 3.");
    if (Ainv != nullptr)
    {
        ACROBATIC_ASSERT(Ainv->IsInitialized() && Ainv->GetRank() == rank, "Can't BatchMatrixInverse with mismatched ranks for Ainv and A.");
        for (int d = 0; d < rank; ++d) ACROBATIC_ASSERT(Ainv->GetDim(d) == A.GetDim(d), "Can't BatchMatrixInverse with mismatched dims for Ainv and A.");
    }
    if (Adet != nullptr)
    {
        ACROBATIC_ASSERT(rank >= 3, "Can't BatchMatrixDet a tensor of rank < 3.");
        ACROBATIC_ASSERT(Adet->IsInitialized() && Adet->GetRank() == rank - 2, "Can't BatchMatrixDet with mismatched ranks for Adet and A.");
        for (int d = 0; d < rank - 2; ++d) ACROBATIC_ASSERT(Adet->GetDim(d) == A.GetDim(d), "Can't BatchMatrixDet with mismatched dims for Adet and A.");
    }
}
}

void TensorEngine::BatchMatrixInverse(Tensor &Ainv, Tensor &A)
{
    check_matrix_batch(A, &Ainv, nullptr);
    RequireCuda("BatchMatrixInverse");
    A.MoveToGPU();
    if (&Ainv != &A) Ainv.SwitchToGPU();
    const int dim = A.GetDim(A.GetRank() - 1);
    check_abi(acro_b200_batch_inv_det(A.GetDeviceData(), Ainv.GetDeviceData(), nullptr, A.GetSize64() / (dim * dim), dim, Stream()),
              "batch_inv_det");
}

void TensorEngine::BatchMatrixDet(Tensor &Adet, Tensor &A)
{
    check_matrix_batch(A, nullptr, &Adet);
    RequireCuda("BatchMatrixDet");
    A.MoveToGPU();
    Adet.SwitchToGPU();
    const int dim = A.GetDim(A.GetRank() - 1);
    check_abi(acro_b200_batch_inv_det(A.GetDeviceData(), nullptr, Adet.GetDeviceData(), A.GetSize64() / (dim * dim), dim, Stream()),
              "batch_inv_det");
}

void TensorEngine::BatchMatrixInvDet(Tensor &Ainv, Tensor &Adet, Tensor &A)
{
    check_matrix_batch(A, &Ainv, &Adet);
    RequireCuda("BatchMatrixInvDet");
    A.MoveToGPU();
    if (&Ainv != &A) Ainv.SwitchToGPU();
    Adet.SwitchToGPU();
    const int dim = A.GetDim(A.GetRank() - 1);
    check_abi(acro_b200_batch_inv_det(A.GetDeviceData(), Ainv.GetDeviceData(), Adet.GetDeviceData(), A.GetSize64() / (dim * dim), dim, Stream()),
              "batch_inv_det");
}

void TensorEngine::FlatIndexedScatter(Tensor &Aout, Tensor &Ain, IndexMapping &M)
{
    ACROBATIC_ASSERT(Aout.IsInitialized() && Ain.IsInitialized(), "FlatIndexedScatter on an uninitialized tensor.");
    ACROBATIC_ASSERT(Aout.GetSize64() == M.GetRangeSize(), "IndexMapping RangeSize does not match the output Tensor size.");
    ACROBATIC_ASSERT(Ain.GetSize64() == M.GetDomainSize(), "IndexMapping DomainSize does not match the input Tensor size.");
    RequireCuda("FlatIndexedScatter");
    Aout.SwitchToGPU();
    Ain.MoveToGPU();
    M.MoveToGPU();
    check_abi(acro_b200_flat_scatter(Aout.GetDeviceData(), Ain.GetDeviceData(), M.GetMap().GetDeviceData(), M.GetRangeSize(), Stream()),
              "flat_scatter");
}

void TensorEngine::FlatIndexedSumGather(Tensor &Aout, Tensor &Ain, IndexMapping &M)
{
    ACROBATIC_ASSERT(Aout.IsInitialized() && Ain.IsInitialized(), "FlatIndexedSumGather on an uninitialized tensor.");
    ACROBATIC_ASSERT(Aout.GetSize64() == M.GetDomainSize(), "IndexMapping DomainSize does not match the output Tensor size.");
    ACROBATIC_ASSERT(Ain.GetSize64() == M.GetRangeSize(), "IndexMapping RangeSize does not match the input Tensor size.");
    RequireCuda("FlatIndexedSumGather");
    if (!M.IsInverseComputed()) M.ComputeInverse();
    Aout.SwitchToGPU();
    Ain.MoveToGPU();
    M.MoveToGPU();
    check_abi(acro_b200_flat_sum_gather(Aout.GetDeviceData(), Ain.GetDeviceData(), M.GetInvMap().GetDeviceData(),
                                        M.GetInvMapOffsets().GetDeviceData(), M.GetDomainSize(), Stream()),
              "flat_sum_gather");
}

void TensorEngine::FlatIndexedSumGather(Tensor &Aout, Tensor &Ain, IndexMapping &M, void *halo)
{
    ACROBATIC_ASSERT(halo != nullptr, "FlatIndexedSumGather over a sharded range needs a shared-entry exchange.");
    FlatIndexedSumGather(Aout, Ain, M);
    check_abi(acro_b200_halo_exchange_sum(static_cast<acro_b200_halo *>(halo), Aout.GetDeviceData(), Stream()), "halo_exchange_sum");
}

namespace
{
// Device memory of one call, handed out and taken back in the order of its stream: calls on other streams, and other captured
// graphs, have their own.
class StreamScratch
{
    public:
    StreamScratch(size_t bytes, void *stream) : Stream(static_cast<cudaStream_t>(stream)), Data(nullptr), Bytes(bytes)
    {
        if (bytes > 0) acroCudaErrorCheck(cudaMallocAsync(&Data, bytes, Stream));
    }
    ~StreamScratch()
    {
        if (Data != nullptr) cudaFreeAsync(Data, Stream);
    }
    StreamScratch(const StreamScratch &) = delete;
    StreamScratch &operator=(const StreamScratch &) = delete;
    void *Get() { return Data; }
    size_t Size() { return Bytes; }

    private:
    cudaStream_t Stream;
    void *Data;
    size_t Bytes;
};

// Tensors that a call overwrites whole (null ones aside).  They stay on the side where they are until the call has been accepted, so that a refused
// one leaves their values where the caller has them; a part of a larger tensor brings the rest of it along, which the call leaves as it is.
class Results
{
    public:
    Results(std::initializer_list<Tensor *> tensors) : Tensors(tensors)
    {
        for (Tensor *T : Tensors)
        {
            if (T == nullptr || T->IsOnGPU()) continue;
            if (dynamic_cast<SliceTensor *>(T) != nullptr) T->MoveToGPU();
            else if (!T->IsMappedToGPU()) T->MapToGPU();
        }
    }
    void Written()
    {
        for (Tensor *T : Tensors)
            if (T != nullptr) T->SwitchToGPU();
    }

    private:
    std::vector<Tensor *> Tensors;
};

void require_shape(Tensor &T, std::initializer_list<int> dims, const char *what)
{
    bool same = T.IsInitialized() && T.GetRank() == static_cast<int>(dims.size());
    int d = 0;
    for (int n : dims) same = same && T.GetDim(d++) == n;
    ACROBATIC_ASSERT(same, std::string("Mismatched dims for ") + what + ".");
}

// Dims of Q, K, V: [sequences][tokens][heads][columns], or without the first.
struct HeadDims
{
    int lead, sequences, tokens, heads, columns;
    HeadDims(Tensor &T, const char *what)
    {
        ACROBATIC_ASSERT(T.IsInitialized() && (T.GetRank() == 3 || T.GetRank() == 4), std::string(what) + " needs 3 or 4 dims.");
        lead = T.GetRank() - 3;
        sequences = lead ? T.GetDim(0) : 1;
        tokens = T.GetDim(lead);
        heads = T.GetDim(lead + 1);
        columns = T.GetDim(lead + 2);
        ACROBATIC_ASSERT(lead == 1 || !T.IsSharded(), std::string(what) + " is one sequence: it cannot be sharded over its tokens.");
    }
    acro_b200_token_array Rows(Tensor &T) const
    {
        const int64_t row = static_cast<int64_t>(heads) * columns;
        return {T.GetDeviceData(), row * tokens, row, columns};
    }
    void Require(Tensor &T, int cols, const char *what) const
    {
        if (lead) require_shape(T, {sequences, tokens, heads, cols}, what);
        else require_shape(T, {tokens, heads, cols}, what);
    }
};

acro_b200_linear_attention_desc attention_desc(const HeadDims &q, const HeadDims &k, const HeadDims &v, double scale)
{
    ACROBATIC_ASSERT(q.lead == k.lead && q.lead == v.lead && q.sequences == k.sequences && q.sequences == v.sequences && q.tokens == k.tokens &&
                         q.tokens == v.tokens && q.columns == k.columns && k.heads == v.heads,
                     "Linear attention with mismatched dims of Q, K and V.");
    acro_b200_linear_attention_desc d = {};
    d.type = ACRO_B200_F64;
    d.q_heads = q.heads;
    d.kv_heads = k.heads;
    d.dk = q.columns;
    d.dv = v.columns;
    d.sequences = q.sequences;
    d.tokens = q.tokens;
    d.scale = scale;
    return d;
}

void require_state(Tensor *S, const HeadDims &q, int dv, const char *what)
{
    if (S == nullptr) return;
    if (q.lead) require_shape(*S, {q.sequences, q.heads, q.columns, dv}, what);
    else require_shape(*S, {q.heads, q.columns, dv}, what);
}

double *device_data(Tensor *T) { return T != nullptr ? T->GetDeviceData() : nullptr; }
}

void TensorEngine::LinearAttention(Tensor &Out, Tensor &Q, Tensor &K, Tensor &V, Tensor &LogDecay, double scale, Tensor *InitialState, Tensor *FinalState)
{
    const HeadDims q(Q, "Q"), k(K, "K"), v(V, "V");
    const acro_b200_linear_attention_desc d = attention_desc(q, k, v, scale);
    q.Require(Out, v.columns, "Out");
    require_shape(LogDecay, {q.heads}, "LogDecay");
    require_state(InitialState, q, v.columns, "InitialState");
    require_state(FinalState, q, v.columns, "FinalState");
    RequireCuda("LinearAttention");
    for (Tensor *T : {&Q, &K, &V, &LogDecay, InitialState})
        if (T != nullptr) T->MoveToGPU();
    Results results({&Out, FinalState});
    HeadDims o = q;
    o.columns = v.columns;
    const acro_b200_token_array rq = q.Rows(Q), rk = k.Rows(K), rv = v.Rows(V), ro = o.Rows(Out);
    StreamScratch scratch(acro_b200_linear_attention_scratch_bytes(&d, 0), Stream());
    check_abi(acro_b200_linear_attention(&d, &rq, &rk, &rv, &ro, LogDecay.GetDeviceData(), nullptr, device_data(InitialState), device_data(FinalState),
                                         nullptr, d.sequences, scratch.Get(), scratch.Size(), Stream()),
              "linear_attention");
    results.Written();
}

void TensorEngine::LinearAttentionStep(Tensor &Out, Tensor &StateOut, Tensor &Q, Tensor &K, Tensor &V, Tensor &LogDecay, Tensor &StateIn, double scale)
{
    ACROBATIC_ASSERT(Q.IsInitialized() && K.IsInitialized() && V.IsInitialized() && Q.GetRank() == 3 && K.GetRank() == 3 && V.GetRank() == 3,
                     "A step of linear attention needs Q, K and V of 3 dims.");
    const int n = Q.GetDim(0), heads = Q.GetDim(1), dk = Q.GetDim(2), kv = K.GetDim(1), dv = V.GetDim(2);
    require_shape(K, {n, kv, dk}, "K");
    require_shape(V, {n, kv, dv}, "V");
    require_shape(Out, {n, heads, dv}, "Out");
    require_shape(LogDecay, {heads}, "LogDecay");
    require_shape(StateIn, {n, heads, dk, dv}, "StateIn");
    require_shape(StateOut, {n, heads, dk, dv}, "StateOut");
    RequireCuda("LinearAttentionStep");
    for (Tensor *T : {&Q, &K, &V, &LogDecay, &StateIn}) T->MoveToGPU();
    Results results({&Out, &StateOut});
    acro_b200_linear_attention_desc d = {};
    d.type = ACRO_B200_F64;
    d.q_heads = heads;
    d.kv_heads = kv;
    d.dk = dk;
    d.dv = dv;
    d.sequences = n;
    d.tokens = 1;
    d.scale = scale;
    const auto rows = [](Tensor &T, int64_t h, int64_t c) { return acro_b200_token_array{T.GetDeviceData(), h * c, h * c, c}; };
    const acro_b200_token_array rq = rows(Q, heads, dk), rk = rows(K, kv, dk), rv = rows(V, kv, dv), ro = rows(Out, heads, dv);
    check_abi(acro_b200_linear_attention_step(&d, &rq, &rk, &rv, &ro, LogDecay.GetDeviceData(), StateIn.GetDeviceData(), StateOut.GetDeviceData(), nullptr,
                                              n, Stream()),
              "linear_attention_step");
    results.Written();
}

void TensorEngine::LinearAttentionBackward(Tensor &dQ, Tensor &dK, Tensor &dV, Tensor &dOut, Tensor &Q, Tensor &K, Tensor &V, Tensor &LogDecay, double scale,
                                           Tensor *InitialState, Tensor *dFinalState, Tensor *dInitialState)
{
    const HeadDims q(Q, "Q"), k(K, "K"), v(V, "V");
    const acro_b200_linear_attention_desc d = attention_desc(q, k, v, scale);
    q.Require(dOut, v.columns, "dOut");
    q.Require(dQ, q.columns, "dQ");
    k.Require(dK, k.columns, "dK");
    v.Require(dV, v.columns, "dV");
    require_shape(LogDecay, {q.heads}, "LogDecay");
    require_state(InitialState, q, v.columns, "InitialState");
    require_state(dFinalState, q, v.columns, "dFinalState");
    require_state(dInitialState, q, v.columns, "dInitialState");
    RequireCuda("LinearAttentionBackward");
    for (Tensor *T : {&Q, &K, &V, &LogDecay, &dOut, InitialState, dFinalState})
        if (T != nullptr) T->MoveToGPU();
    Results results({&dQ, &dK, &dV, dInitialState});
    HeadDims o = q;
    o.columns = v.columns;
    const acro_b200_token_array rq = q.Rows(Q), rk = k.Rows(K), rv = v.Rows(V), ro = o.Rows(dOut), gq = q.Rows(dQ), gk = k.Rows(dK), gv = v.Rows(dV);
    StreamScratch scratch(acro_b200_linear_attention_backward_scratch_bytes(&d, 0), Stream());
    check_abi(acro_b200_linear_attention_backward(&d, &rq, &rk, &rv, &ro, LogDecay.GetDeviceData(), nullptr, device_data(InitialState),
                                                  device_data(dFinalState), &gq, &gk, &gv, device_data(dInitialState), scratch.Get(), scratch.Size(),
                                                  Stream()),
              "linear_attention_backward");
    results.Written();
}

void TensorEngine::LayerNorm(Tensor &Y, Tensor &X, Tensor *Weight, Tensor *Bias, double eps, Tensor *Mean, Tensor *Rstd)
{
    ACROBATIC_ASSERT(X.IsInitialized() && X.GetRank() >= 1, "LayerNorm needs a tensor of at least one dim.");
    ACROBATIC_ASSERT(X.GetRank() > 1 || !X.IsSharded(), "LayerNorm of a single row that is sharded over its entries.");
    const int width = X.GetDim(X.GetRank() - 1);
    const int64_t rows = X.GetSize64() / width;
    ACROBATIC_ASSERT(Y.IsInitialized() && Y.GetSize64() == X.GetSize64(), "Mismatched sizes of X and Y.");
    for (Tensor *T : {Weight, Bias})
        if (T != nullptr) require_shape(*T, {width}, "Weight or Bias");
    for (Tensor *T : {Mean, Rstd})
        ACROBATIC_ASSERT(T == nullptr || (T->IsInitialized() && T->GetSize64() == rows), "Mean and Rstd have one entry per row.");
    RequireCuda("LayerNorm");
    for (Tensor *T : {&X, Weight, Bias})
        if (T != nullptr) T->MoveToGPU();
    Results results({&Y, Mean, Rstd});
    check_abi(acro_b200_layer_norm(ACRO_B200_F64, X.GetDeviceData(), width, device_data(Weight), device_data(Bias), Y.GetDeviceData(), width, device_data(Mean),
                                   device_data(Rstd), rows, width, eps, Stream()),
              "layer_norm");
    results.Written();
}

void TensorEngine::LayerNormBackward(Tensor &dX, Tensor *dWeight, Tensor *dBias, Tensor &dY, Tensor &X, Tensor &Mean, Tensor &Rstd, Tensor *Weight)
{
    ACROBATIC_ASSERT(X.IsInitialized() && X.GetRank() >= 1, "LayerNormBackward needs a tensor of at least one dim.");
    ACROBATIC_ASSERT(X.GetRank() > 1 || !X.IsSharded(), "LayerNormBackward of a single row that is sharded over its entries.");
    const int width = X.GetDim(X.GetRank() - 1);
    const int64_t rows = X.GetSize64() / width;
    for (Tensor *T : {&dX, &dY}) ACROBATIC_ASSERT(T->IsInitialized() && T->GetSize64() == X.GetSize64(), "Mismatched sizes of X, dX and dY.");
    for (Tensor *T : {Weight, dWeight, dBias})
        if (T != nullptr) require_shape(*T, {width}, "Weight, dWeight or dBias");
    for (Tensor *T : {&Mean, &Rstd}) ACROBATIC_ASSERT(T->IsInitialized() && T->GetSize64() == rows, "Mean and Rstd have one entry per row.");
    RequireCuda("LayerNormBackward");
    for (Tensor *T : {&dY, &X, &Mean, &Rstd, Weight})
        if (T != nullptr) T->MoveToGPU();
    Results results({&dX, dWeight, dBias});
    const bool sums = dWeight != nullptr || dBias != nullptr;
    StreamScratch scratch(sums ? acro_b200_layer_norm_backward_scratch_bytes(ACRO_B200_F64, rows, width) : 0, Stream());
    check_abi(acro_b200_layer_norm_backward(ACRO_B200_F64, dY.GetDeviceData(), width, X.GetDeviceData(), width, device_data(Weight), Mean.GetDeviceData(),
                                            Rstd.GetDeviceData(), dX.GetDeviceData(), width, device_data(dWeight), device_data(dBias), rows, width,
                                            scratch.Get(), scratch.Size(), Stream()),
              "layer_norm_backward");
    results.Written();
    if (ThePeerGroup == nullptr || !X.IsSharded()) return;
    for (Tensor *T : {dWeight, dBias})
        if (T != nullptr)
            check_abi(acro_b200_peer_allreduce(T->GetDeviceData(), T->GetDeviceData(), width, ACRO_B200_OP_ASSIGN,
                                               static_cast<acro_b200_peer_group *>(ThePeerGroup), Stream()),
                      "peer_allreduce");
}

TensorKernel *TensorEngine::GetAddTensorKernel(std::string &kernel_str)
{
    auto it = KernelMap.find(kernel_str);
    if (it == KernelMap.end())
    {
        it = KernelMap.emplace(kernel_str, std::unique_ptr<TensorKernel>(new TensorKernel(kernel_str))).first;
    }
    return it->second.get();
}

DimensionedKernel *TensorEngine::GetAddDimensionedKernel(TensorKernel *kernel, Tensor *output, std::vector<Tensor *> &inputs)
{
    // The key spells the kernel and every loop extent, so equal keys mean equal bindings.
    std::string key = kernel->GetDimensionedNameString(output, inputs);
    auto it = DimensionedKernelMap.find(key);
    if (it == DimensionedKernelMap.end())
    {
        it = DimensionedKernelMap.emplace(key, std::unique_ptr<DimensionedKernel>(new DimensionedKernel(kernel, output, inputs))).first;
    }
    return it->second.get();
}

KernelExecutor *TensorEngine::GetAddKernelExecutor()
{
    std::string key;
    for (DimensionedKernel *k : MKLKernels) key += k->GetDimensionedNameString() + ";";
    auto it = ExecutorMap.find(key);
    if (it == ExecutorMap.end())
    {
        KernelExecutor *executor = KernelExecutor::Create(ExecutorType, new DimensionedMultiKernel(MKLKernels));
        it = ExecutorMap.emplace(key, std::unique_ptr<KernelExecutor>(executor)).first;
    }
    return it->second.get();
}

}
