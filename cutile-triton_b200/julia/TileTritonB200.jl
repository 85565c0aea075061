"""
    TileTritonB200

B200 (sm_100a) backend for TileTriton: the same user-facing API as
`TritonRun` / `TritonShim` (reference: src/runtime.jl, src/shim.jl), with the
TTIR -> Triton -> cubin pipeline replaced by prebuilt kernels in
`libcutile_b200.so`, reached through `ccall` on the C ABI declared in
include/cutile_b200.h.

- `triton_kernel(f, argtypes; name, num_warps, num_stages, use_tma)` returns a
  `B200Kernel` handle (no compilation; unknown kernels raise).
- `launch!(k, grid, args...)` flattens exactly like `TritonRun.flatten_args`
  (runtime.jl:163-198) into `ctb_array`s and launches on CUDA.jl's stream.
- `install_shim!()` overwrites `cuTile.cufunction` so `ct.launch` /
  `@cuda backend=cuTile` of the registered kernels run here (shim.jl:126-131).
- `use_b200!()` selects this backend for `TileTriton.triton_kernel` /
  `launch!` callers (TileTriton's own `triton_kernel`/`launch!` forward here
  when the active target's backend is "b200").

The library path is `ENV["CUTILE_B200_LIB"]`, else the in-tree build.
"""
module TileTritonB200

using CUDA
using Libdl
import cuTile as ct

export triton_kernel, triton_kernel_candidates, launch!, install_shim!, use_b200!, B200Kernel,
       softmax_host!, layernorm_fwd_host!, vadd_host!, moe_align,
       dense!, dense_bwd!, moe_route, moe_route_bwd, moe_combine!, moe_combine_bwd

# ---------------------------------------------------------------------------- library
const LIBPATH = Ref{String}("")
const LIB = Ref{Ptr{Cvoid}}(C_NULL)
const SYMS = Dict{Symbol,Ptr{Cvoid}}()

default_libpath() = get(ENV, "CUTILE_B200_LIB",
                        normpath(joinpath(@__DIR__, "..", "cutile_b200", "libcutile_b200.so")))

function sym(name::Symbol)
    if LIB[] == C_NULL
        LIBPATH[] = default_libpath()
        isfile(LIBPATH[]) || error("b200: libcutile_b200.so not found at $(LIBPATH[])")
        LIB[] = Libdl.dlopen(LIBPATH[])
    end
    get!(() -> Libdl.dlsym(LIB[], name), SYMS, name)
end

lasterror() = unsafe_string(ccall(sym(:ctb_last_error), Cstring, ()))
check(rc::Integer) = rc == 0 ? nothing : error("b200: " * lasterror())

# ---------------------------------------------------------------------------- ABI types
const CTB_MAX_DIMS = 5

"`ctb_array`: one flattened TileArray (pointer, Julia-order sizes and strides)."
struct CtbArray
    ptr::Ptr{Cvoid}
    ndim::Int32
    dtype::Int32
    sizes::NTuple{CTB_MAX_DIMS,Int32}
    strides::NTuple{CTB_MAX_DIMS,Int32}
end

struct CtbKernelInfo
    name::NTuple{32,UInt8}
    narrays::Int32
    nscalars::Int32
    num_warps::Int32
    shared_bytes::Int32
end

dtype_code(::Type{Float16}) = Int32(1)
dtype_code(::Type{Float32}) = Int32(3)
dtype_code(::Type{Float64}) = Int32(4)
dtype_code(::Type{Int32}) = Int32(5)
dtype_code(T::Type) = T === ct.TFloat32 ? error("b200: tf32 inputs are stored as Float32 arrays") :
                      (nameof(T) === :BFloat16 ? Int32(2) : error("b200: unsupported element type $T"))

pad5(t) = ntuple(i -> i <= length(t) ? Int32(t[i]) : Int32(0), CTB_MAX_DIMS)

ctb_array(a::CuArray{T,N}) where {T,N} =
    CtbArray(reinterpret(Ptr{Cvoid}, UInt(pointer(a))), Int32(N), dtype_code(T),
             pad5(size(a)), pad5(strides(a)))

# A converted cuTile argument (what ShimKernel receives; shim.jl:42-63).
ctb_array(x::ct.TileArray) =
    CtbArray(reinterpret(Ptr{Cvoid}, UInt(x.ptr)), Int32(length(x.sizes)),
             dtype_code(eltype(x)), pad5(x.sizes), pad5(x.strides))

# ---------------------------------------------------------------------------- kernels
"Per-parameter ABI record (the reference ArgSpec, src/emitter.jl:163-167)."
struct B200ArgSpec
    kind::Symbol      # :tilearray | :scalar
    elty::Type
    ndims::Int
end

"A prebuilt-kernel handle (the TritonKernel analogue, runtime.jl:85-95)."
struct B200Kernel
    handle::Int32
    name::String
    num_warps::Int
    warp_size::Int
    shared::Int
    global_scratch_size::Int
    argspec::Vector{B200ArgSpec}
end

function argspec_of(argtypes::Type{<:Tuple})
    specs = B200ArgSpec[]
    consts = Int64[]
    for T in argtypes.parameters
        if T <: ct.TileArray
            push!(specs, B200ArgSpec(:tilearray, eltype(T), ndims(T)))
        elseif T <: ct.Constant
            push!(consts, Int64(T.parameters[2]))   # Constant{Int, V}: ghost
        else
            push!(specs, B200ArgSpec(:scalar, T, 0))
        end
    end
    return specs, consts
end

"""
    triton_kernel(f, argtypes; name, num_warps, num_stages, use_tma) -> B200Kernel

Looks up the prebuilt sm_100a kernel for cuTile function `f`. The keyword
arguments are accepted for signature compatibility with
`TritonRun.triton_kernel`; the schedule of each kernel is fixed.
"""
function triton_kernel(@nospecialize(f), @nospecialize(argtypes); name::String=string(nameof(f)),
                       num_warps=nothing, num_stages=nothing, use_tma::Bool=true)
    specs, consts = argspec_of(argtypes)
    dts = Int32[dtype_code(s.elty) for s in specs if s.kind === :tilearray]
    h = Ref{Int32}(-1)
    kname = string(nameof(f))
    check(ccall(sym(:ctb_find_kernel), Cint,
                (Cstring, Ptr{Int32}, Int32, Ptr{Int64}, Int32, Ref{Int32}),
                kname, dts, length(dts), consts, length(consts), h))
    info = Ref{CtbKernelInfo}()
    check(ccall(sym(:ctb_kernel_info_get), Cint, (Int32, Ref{CtbKernelInfo}), h[], info))
    nscal = count(s -> s.kind === :scalar, specs)
    nscal == info[].nscalars ||
        error("b200: $kname expects $(info[].nscalars) scalar parameters, got $nscal")
    return B200Kernel(h[], kname, info[].num_warps, 32, info[].shared_bytes, 0, specs)
end

"One candidate: the hand-written kernel has no variants to race."
triton_kernel_candidates(@nospecialize(f), @nospecialize(argtypes); name::String=string(nameof(f)),
                         use_tma::Bool=true) = [triton_kernel(f, argtypes; name, use_tma)]

function flatten_args(spec::Vector{B200ArgSpec}, args)
    length(spec) == length(args) || error("expected $(length(spec)) kernel arguments")
    arrays = CtbArray[]
    scalars = Float64[]
    for (s, a) in zip(spec, args)
        if s.kind === :tilearray
            a isa AbstractArray || a isa ct.TileArray || error("expected a GPU array for tilearray argument")
            eltype(a) === s.elty || error("eltype mismatch: $(eltype(a)) vs $(s.elty)")
            (a isa ct.TileArray ? length(a.sizes) : ndims(a)) == s.ndims || error("ndims mismatch")
            push!(arrays, ctb_array(a))
        else
            push!(scalars, Float64(a))
        end
    end
    return arrays, scalars
end

function raw_launch(handle::Int32, arrays::Vector{CtbArray}, scalars::Vector{Float64}, g)
    grid = Int32[g[1], g[2], g[3]]
    rc = ccall(sym(:ctb_launch), Cint,
               (Int32, Ptr{CtbArray}, Int32, Ptr{Float64}, Int32, Ptr{Int32}, Ptr{Cvoid}),
               handle, arrays, length(arrays), scalars, length(scalars), grid,
               CUDA.stream().handle)
    check(rc)
end

normgrid(grid) = grid isa Integer ? (Int(grid), 1, 1) :
                 length(grid) == 2 ? (grid[1], grid[2], 1) : Tuple(grid)

"""
    launch!(k::B200Kernel, grid, args...)

`grid` is advisory (outputs never depend on it); `args` are the kernel's
Julia-level arguments in order, skipping `ct.Constant` slots.
"""
function launch!(k::B200Kernel, grid, args...)
    arrays, scalars = flatten_args(k.argspec, args)
    GC.@preserve args raw_launch(k.handle, arrays, scalars, normgrid(grid))
    return nothing
end

# ---------------------------------------------------------------------------- shim
mutable struct B200ShimKernel{F,TT} <: ct.AbstractKernel{F,TT}
    kernel::B200Kernel
    f::F
end

const KERNEL_CACHE = Dict{Any,Any}()

function get_kernel(@nospecialize(f), @nospecialize(tt))
    key = (f, tt, Base.get_world_counter())
    haskey(KERNEL_CACHE, key) && return KERNEL_CACHE[key]
    k = B200ShimKernel{typeof(f),tt}(triton_kernel(f, tt), f)
    KERNEL_CACHE[key] = k
    return k
end

# Ghost arguments (Constant and other singletons) carry no bytes; dropping them
# with a recursive tuple filter is specialised per signature, with no Any[].
drop_ghosts() = ()
drop_ghosts(a, rest...) = Base.issingletontype(typeof(a)) ? drop_ghosts(rest...) :
                          (a, drop_ghosts(rest...)...)

# cuTile calls the kernel with converted arguments (TileArrays, ghosts, primitives).
function (k::B200ShimKernel)(args...; blocks=1, threads=1, convert=Val(false), kwargs...)
    arrays, scalars = flatten_args(k.kernel.argspec, drop_ghosts(args...))
    GC.@preserve args raw_launch(k.kernel.handle, arrays, scalars, normgrid(blocks))
    return nothing
end

"""
    install_shim!()

Route cuTile compilation of the registered kernels to libcutile_b200.so by
overwriting `cuTile.cufunction` (opt-in, like the reference's shim).
"""
function install_shim!()
    @eval ct function cufunction(@nospecialize(f), tt::Type{<:Tuple}=Tuple{}; kwargs...)
        return $(TileTritonB200).get_kernel(f, tt)
    end
    return nothing
end

# ---- host-buffer calls: arrays in (pinned) host memory, chunks pipelined through
# a device workspace on the library's streams; synchronise the stream to read results.
const HOST_WS = Ref{Any}(nothing)
function host_workspace(nbytes::Integer)
    ws = HOST_WS[]
    if ws === nothing || sizeof(ws) < nbytes
        ws = CuArray{UInt8}(undef, max(Int(nbytes), 256))
        HOST_WS[] = ws
    end
    return ws
end
wsbytes(inb, outb, units) = ccall(sym(:ctb_host_workspace_bytes), Int64, (Int64, Int64, Int64),
                                  inb, outb, units)

"y = softmax over each column of the host matrix x (len x count), through the GPU."
function softmax_host!(y::Matrix{Float32}, x::Matrix{Float32})
    len, count = size(x)
    ws = host_workspace(wsbytes(4len, 4len, count))
    check(ccall(sym(:ctb_softmax_f32_host), Cint,
                (Ptr{Float32}, Ptr{Float32}, Int32, Int32, CuPtr{UInt8}, Int64, Ptr{Cvoid}),
                x, y, len, count, ws, sizeof(ws), CUDA.stream().handle))
    CUDA.synchronize()
    return y
end

"LayerNorm over each column of the host matrix x (n x rows): y, mean, rstd on the host."
function layernorm_fwd_host!(y::Matrix{Float32}, mean::Vector{Float32}, rstd::Vector{Float32},
                             x::Matrix{Float32}, w::Vector{Float32}, b::Vector{Float32}, eps=1f-5)
    n, rows = size(x)
    ws = host_workspace(wsbytes(4n, 4n + 8, rows) + 2 * cld(4n, 256) * 256)
    check(ccall(sym(:ctb_layernorm_fwd_f32_host), Cint,
                (Ptr{Float32}, Ptr{Float32}, Ptr{Float32}, Ptr{Float32}, Ptr{Float32}, Ptr{Float32},
                 Int32, Int32, Float32, CuPtr{UInt8}, Int64, Ptr{Cvoid}),
                x, w, b, y, mean, rstd, n, rows, eps, ws, sizeof(ws), CUDA.stream().handle))
    CUDA.synchronize()
    return y, mean, rstd
end

"c = a + b for host vectors, through the GPU."
function vadd_host!(c::Vector{T}, a::Vector{T}, b::Vector{T}) where {T<:Union{Float16,Float32,Float64}}
    ws = host_workspace(wsbytes(2sizeof(T), sizeof(T), length(a)) + 16 * 256)
    check(ccall(sym(:ctb_vadd_host), Cint,
                (Int32, Ptr{T}, Ptr{T}, Ptr{T}, Int64, CuPtr{UInt8}, Int64, Ptr{Cvoid}),
                dtype_code(T), a, b, c, length(a), ws, sizeof(ws), CUDA.stream().handle))
    CUDA.synchronize()
    return c
end

"""
    moe_align(topk_ids::Matrix{<:Integer}, num_experts; block=256)

Fused-MoE routing for the `moe` kernel from a (topk, tokens) matrix of
0-based expert ids: (sorted_token_ids, expert_ids, num_tokens_post_padded) as
Int32 vectors, slots grouped by expert in slot order, each expert padded to a
multiple of `block` (256: CTA-pair kernel, 128: single-SM kernel) with the id
tokens*topk. Move them to the device with `CuArray`.
"""
function moe_align(topk_ids::AbstractMatrix{<:Integer}, num_experts::Integer; block::Integer=256)
    flat = vec(topk_ids)  # slot s = token * topk + choice (column-major (topk, tokens))
    n = length(flat)
    sorted = Int32[]
    experts = Int32[]
    for e in 0:num_experts-1
        slots = [Int32(s - 1) for s in 1:n if flat[s] == e]
        pad = mod(-length(slots), block)
        append!(sorted, slots, fill(Int32(n), pad))
        append!(experts, fill(Int32(e), (length(slots) + pad) ÷ block))
    end
    em = length(sorted)
    if em == 0  # nothing routed: one padding block with no expert, none in use
        sorted = fill(Int32(n), block)
        experts = Int32[-1]
    end
    return sorted, experts, Int32[em]
end

"""
    moe_align(topk_ids::CuMatrix{Int32}, num_experts; block=256)

The same routing on the device (`ctb_moe_align_i32`), with no host round trip:
the outputs are CuArrays sized for the worst case (`ctb_moe_align_capacity`);
entries past num_tokens_post_padded hold the padding id and blocks past it the
expert -1, which the `moe` kernel skips. At most 256 experts.
"""
function moe_align(topk_ids::CuMatrix{Int32}, num_experts::Integer; block::Integer=256)
    n = length(topk_ids)
    cap = ccall(sym(:ctb_moe_align_capacity), Int32, (Int32, Int32, Int32), n, num_experts, block)
    cap < 0 && error("b200: moe_align: bad sizes")
    sorted = CuArray{Int32}(undef, cap)
    experts = CuArray{Int32}(undef, cap ÷ block)
    ntp = CuArray{Int32}(undef, 1)
    check(ccall(sym(:ctb_moe_align_i32), Cint,
                (CuPtr{Int32}, Int32, Int32, Int32, CuPtr{Int32}, CuPtr{Int32}, CuPtr{Int32},
                 Int32, Ptr{Cvoid}),
                topk_ids, n, num_experts, block, sorted, experts, ntp, cap,
                CUDA.stream().handle))
    return sorted, experts, ntp
end

# ---------------------------------------------------------------------------- layer calls
const ACTS = Dict(:none => 0, :relu => 1, :gelu => 2, :gelu_tanh => 3, :silu => 4)
const SCORES = Dict(:softmax => 0, :sigmoid => 1)
# The column stride that the C ABI is given; one column has none that matters.
ldim(x) = size(x, 2) > 1 ? stride(x, 2) : max(size(x, 1), 1)
ldor0(x) = x === nothing ? 0 : ldim(x)
orC(x) = x === nothing ? CU_NULL : pointer(x)

"""
    operand(x, what, T, dims; packed=false)

What the library cannot see in a pointer: that `x` (or `nothing`) is a device
array of element type `T` and size `dims` whose columns are contiguous, and with
`packed` follow one another.
"""
function operand(x, what::String, T::Type, dims::Dims; packed::Bool=false)
    x === nothing && return nothing
    x isa StridedCuArray || error("b200: $what: expected a device array, got $(typeof(x))")
    eltype(x) === T || error("b200: $what: expected elements of type $T, got $(eltype(x))")
    size(x) == dims || error("b200: $what: expected size $dims, got $(size(x))")
    size(x, 1) <= 1 || stride(x, 1) == 1 || error("b200: $what: columns must be contiguous")
    packed && length(dims) == 2 && ldim(x) != max(dims[1], 1) && error("b200: $what: must be contiguous")
    return nothing
end

# The 16-bit types of the layer calls. BFloat16 is known by its name: it is Core's
# from Julia 1.11 on and a package's before.
function layer_code(what::String, T::Type)
    c = dtype_code(T)
    c == 1 || c == 2 || error("b200: $what: matrices must be Float16 or BFloat16, got $T")
    return c
end
choice(table, key::Symbol, what::String) =
    get(() -> error("b200: $what: none of $(join(keys(table), ", "))"), table, key)

"""
    dense!(C, A, B; bias=nothing, act=:none, R=nothing, Z=nothing)

C = act.(A * B .+ bias) .+ R for Float16 or BFloat16 columns: A (M, K) the
weight, B (K, N) a column per token; `act` one of :none, :relu, :gelu,
:gelu_tanh, :silu; bias of the matrices' type or Float32; Z receives the value
before the activation (`ctb_dense_fwd`).
"""
function dense!(C::StridedCuMatrix{T}, A::StridedCuMatrix{T}, B::StridedCuMatrix{T}; bias=nothing,
                act::Symbol=:none, R=nothing, Z=nothing) where {T}
    code = layer_code("dense!", T)
    M, K = size(A)
    N = size(B, 2)
    operand(A, "dense!: A", T, (M, K))
    operand(B, "dense!: B", T, (K, N))
    operand(C, "dense!: C", T, (M, N))
    operand(bias, "dense!: bias", bias isa AbstractArray{Float32} ? Float32 : T, (M,))
    operand(R, "dense!: R", T, (M, N))
    operand(Z, "dense!: Z", T, (M, N))
    a = choice(ACTS, act, "dense!: act")
    nws = ccall(sym(:ctb_dense_fwd_workspace_bytes), Int64,
                (CuPtr{T}, CuPtr{T}, Int32, Int32, Int32, Int64, Int64), A, B, M, N, K, ldim(A), ldim(B))
    ws = CuArray{UInt8}(undef, max(nws, 1))
    GC.@preserve A B C bias R Z ws check(ccall(sym(:ctb_dense_fwd), Cint,
                (Int32, CuPtr{T}, CuPtr{T}, CuPtr{Cvoid}, Int32, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{T},
                 Int32, Int32, Int32, Int64, Int64, Int64, Int64, Int64, Int32, CuPtr{UInt8}, Int64,
                 Ptr{Cvoid}),
                code, A, B, orC(bias), bias === nothing ? 0 : dtype_code(eltype(bias)), orC(R), orC(Z),
                C, M, N, K, ldim(A), ldim(B), ldor0(R), ldor0(Z), ldim(C), a, ws, nws,
                CUDA.stream().handle))
    return C
end

"""
    dense_bwd!(dA, dB, dbias, dC, A, B; act=:none, Z=nothing)

Gradients of `dense!` from dC (M, N); any of dA (M, K), dB (K, N), dbias (M,
Float32) may be `nothing`. Z is the forward call's (`ctb_dense_bwd`).
"""
function dense_bwd!(dA, dB, dbias, dC::StridedCuMatrix{T}, A::StridedCuMatrix{T}, B::StridedCuMatrix{T};
                    act::Symbol=:none, Z=nothing) where {T}
    code = layer_code("dense_bwd!", T)
    M, K = size(A)
    N = size(B, 2)
    operand(dC, "dense_bwd!: dC", T, (M, N))
    operand(A, "dense_bwd!: A", T, (M, K))
    operand(B, "dense_bwd!: B", T, (K, N))
    operand(Z, "dense_bwd!: Z", T, (M, N))
    operand(dA, "dense_bwd!: dA", T, (M, K))
    operand(dB, "dense_bwd!: dB", T, (K, N))
    operand(dbias, "dense_bwd!: dbias", Float32, (M,))
    a = choice(ACTS, act, "dense_bwd!: act")
    nws = ccall(sym(:ctb_dense_bwd_workspace_bytes), Int64,
                (CuPtr{T}, CuPtr{T}, CuPtr{T}, Int32, Int32, Int32, Int64, Int64, Int64, Int32, Int32),
                dC, A, B, M, N, K, ldim(dC), ldim(A), ldim(B), a, dbias === nothing ? 0 : 1)
    ws = CuArray{UInt8}(undef, max(nws, 1))
    GC.@preserve dA dB dbias dC A B Z ws check(ccall(sym(:ctb_dense_bwd), Cint,
                (Int32, CuPtr{T}, CuPtr{T}, CuPtr{T}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid},
                 CuPtr{Cvoid}, Int32, Int32, Int32, Int64, Int64, Int64, Int64, Int64, Int64, Int32,
                 CuPtr{UInt8}, Int64, Ptr{Cvoid}),
                code, dC, A, B, orC(Z), orC(dA), orC(dB), orC(dbias), M, N, K, ldim(dC), ldim(A),
                ldim(B), ldor0(Z), ldor0(dA), ldor0(dB), a, ws, nws, CUDA.stream().handle))
    return dA, dB, dbias
end

"""
    moe_route(logits, topk; score=:softmax, bias, groups=1, topk_groups=groups, group_top=2,
              renorm=true, scale=1) -> (weights, ids)

Routes each column of the (E, T) logits to `topk` experts (`ctb_moe_route`):
weights Float32 and 0-based ids Int32, both (topk, T), for `moe_align` and the
`moe` kernel; id -1 where no expert is available.
"""
function moe_route(logits::StridedCuMatrix{T}, topk::Integer; score::Symbol=:softmax, bias=nothing,
                   groups::Integer=1, topk_groups::Integer=groups, group_top::Integer=2,
                   renorm::Bool=true, scale::Real=1) where {T}
    E, n = size(logits)
    topk >= 1 || error("b200: moe_route: topk must be positive")
    operand(logits, "moe_route: logits", T, (E, n))
    operand(bias, "moe_route: bias", Float32, (E,))
    weights, ids = CuArray{Float32}(undef, topk, n), CuArray{Int32}(undef, topk, n)
    GC.@preserve bias check(ccall(sym(:ctb_moe_route), Cint,
                (Int32, CuPtr{T}, CuPtr{Cvoid}, CuPtr{Float32}, CuPtr{Int32}, Int32, Int32, Int32, Int64,
                 Int32, Int32, Int32, Int32, Int32, Float32, Ptr{Cvoid}),
                dtype_code(T), logits, orC(bias), weights, ids, n, E, topk, ldim(logits),
                choice(SCORES, score, "moe_route: score"), groups, topk_groups, group_top, renorm, scale,
                CUDA.stream().handle))
    return weights, ids
end

"Gradient of `moe_route`'s weights with respect to the logits, for the ids it gave (`ctb_moe_route_bwd`)."
function moe_route_bwd(dweights::CuMatrix{Float32}, logits::StridedCuMatrix{T}, ids::CuMatrix{Int32};
                       score::Symbol=:softmax, renorm::Bool=true, scale::Real=1) where {T}
    E, n = size(logits)
    topk = size(ids, 1)
    operand(logits, "moe_route_bwd: logits", T, (E, n))
    operand(ids, "moe_route_bwd: ids", Int32, (topk, n); packed=true)
    operand(dweights, "moe_route_bwd: dweights", Float32, (topk, n); packed=true)
    dlogits = CuArray{T}(undef, E, n)
    check(ccall(sym(:ctb_moe_route_bwd), Cint,
                (Int32, CuPtr{Float32}, CuPtr{T}, CuPtr{Int32}, CuPtr{T}, Int32, Int32, Int32, Int64, Int64,
                 Int32, Int32, Float32, Ptr{Cvoid}),
                dtype_code(T), dweights, logits, ids, dlogits, n, E, topk, ldim(logits), E,
                choice(SCORES, score, "moe_route_bwd: score"), renorm, scale, CUDA.stream().handle))
    return dlogits
end

"""
    moe_combine!(out, y, topk; weights=nothing, ids=nothing, num_experts=0, R=nothing)

out[:, t] = R[:, t] + sum over j of weights[j, t] * y[:, (t - 1) topk + j], slots
with an id outside 0:num_experts-1 left out (`ctb_moe_combine`).
"""
function moe_combine!(out::StridedCuMatrix{T}, y::StridedCuMatrix{T}, topk::Integer; weights=nothing,
                      ids=nothing, num_experts::Integer=0, R=nothing) where {T}
    code = layer_code("moe_combine!", T)
    N, n = size(out)
    topk >= 1 || error("b200: moe_combine!: topk must be positive")
    operand(out, "moe_combine!: out", T, (N, n))
    operand(y, "moe_combine!: y", T, (N, Int(n * topk)))
    operand(weights, "moe_combine!: weights", Float32, (Int(topk), n); packed=true)
    operand(ids, "moe_combine!: ids", Int32, (Int(topk), n); packed=true)
    operand(R, "moe_combine!: R", T, (N, n))
    GC.@preserve weights ids R check(ccall(sym(:ctb_moe_combine), Cint,
                (Int32, CuPtr{T}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{T}, Int32, Int32, Int32,
                 Int32, Int64, Int64, Int64, Ptr{Cvoid}),
                code, y, orC(weights), orC(ids), orC(R), out, n, topk, N, num_experts, ldim(y), ldor0(R),
                ldim(out), CUDA.stream().handle))
    return out
end

"Gradients (dy, dweights) of `moe_combine!` from dout (N, T) (`ctb_moe_combine_bwd`)."
function moe_combine_bwd(dout::StridedCuMatrix{T}, y, topk::Integer; weights=nothing, ids=nothing,
                         num_experts::Integer=0) where {T}
    code = layer_code("moe_combine_bwd", T)
    N, n = size(dout)
    topk >= 1 || error("b200: moe_combine_bwd: topk must be positive")
    weights === nothing || y !== nothing || error("b200: moe_combine_bwd: weights need y")
    ys = weights === nothing ? nothing : y  # not used without weights
    operand(dout, "moe_combine_bwd: dout", T, (N, n))
    operand(ys, "moe_combine_bwd: y", T, (N, Int(n * topk)))
    operand(weights, "moe_combine_bwd: weights", Float32, (Int(topk), n); packed=true)
    operand(ids, "moe_combine_bwd: ids", Int32, (Int(topk), n); packed=true)
    dy = CuArray{T}(undef, N, n * topk)
    dweights = weights === nothing ? nothing : CuArray{Float32}(undef, topk, n)
    GC.@preserve ys weights ids dweights check(ccall(sym(:ctb_moe_combine_bwd), Cint,
                (Int32, CuPtr{T}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{Cvoid}, CuPtr{T}, CuPtr{Cvoid}, Int32,
                 Int32, Int32, Int32, Int64, Int64, Int64, Ptr{Cvoid}),
                code, dout, orC(ys), orC(weights), orC(ids), dy, orC(dweights), n, topk, N, num_experts,
                ldim(dout), ldor0(ys), max(N, 1), CUDA.stream().handle))
    return dy, dweights
end

"Initialises the library on the active CUDA device (kernel attributes, checks sm_100)."
function use_b200!()
    check(ccall(sym(:ctb_init), Cint, (Cint,), CUDA.deviceid(CUDA.device())))
    @info "TileTriton: using the B200 sm_100a kernel library $(LIBPATH[])"
    return nothing
end

end # module
