{===============================================================================
  Gemma4.Cache - binding of libgemma4_sampler.so's 8-bit cache
  (include/gemma4_cache.h), beside Gemma4.Beam, whose pages it fills and reads.

  As in Gemma4.Sampler, every external has its export's argument order and C
  types, arrays and records are typed pointers passed by value, and a failing
  call of the class adds an esError entry to GetErrors() and returns False.
===============================================================================}

unit Gemma4.Cache;

{$IFDEF FPC}{$MODE DELPHI}{$ENDIF}

interface

uses
  SysUtils,
  StdApp.Base,
  Gemma4.Sampler,
  Gemma4.Beam;

const
  CSM_ERR_CACHE = 'SM07';

  G4S_CACHE_MAX_HEADS = 512;
  G4S_CACHE_MAX_KV_HEADS = 64;
  G4S_CACHE_MAX_GROUP = 64;
  G4S_CACHE_MAX_HEAD_DIM = 512;
  G4S_CACHE_MAX_SCALE_TOKENS = 256;
  G4S_CACHE_MAX_TOKENS = 1048576;
  G4S_CACHE_MAX_CONTEXT = 1073741824;

  G4S_ROTARY_HALVES = 0;
  G4S_ROTARY_NEIGHBOURS = 1;

type
  { PG4SCache }
  // opaque g4s_cache*
  PG4SCache = Pointer;
  PPG4SCache = ^PG4SCache;

  { TG4SCacheConfig }
  TG4SCacheConfig = record
    Heads: Integer;
    KvHeads: Integer;
    HeadDim: Integer;
    ScaleTokens: Integer;
    RotaryDims: Integer;
    RotaryPairs: Integer;
  end;
  PG4SCacheConfig = ^TG4SCacheConfig;

  { TG4SCacheView }
  // head h of token i at Data + (i*TokenStride + h*HeadStride) elements
  TG4SCacheView = record
    Data: Pointer;
    TokenStride: Int64;
    HeadStride: Int64;
  end;
  PG4SCacheView = ^TG4SCacheView;

function g4s_cache_create(AOut: PPG4SCache; AGeometry: PG4SPageGeometry;
  AConfig: PG4SCacheConfig; AHipStream: Pointer): Integer; cdecl; external CG4SLib;
function g4s_cache_destroy(ACache: PG4SCache): Integer; cdecl; external CG4SLib;
function g4s_cache_last_error(ACache: PG4SCache): PAnsiChar; cdecl; external CG4SLib;
function g4s_cache_append(ACache: PG4SCache; AState: PG4SPageState; ARows: Integer;
  ADevStarts: PInteger; ATokens: Integer; ADType: Integer; AQ: PG4SCacheView;
  AK: PG4SCacheView; AV: PG4SCacheView; AQOut: PG4SCacheView; ADevPositions: PInteger;
  ADevFreqs: PSingle; ADevPool: Pointer; AKPlane: Integer; AVPlane: Integer): Integer;
  cdecl; external CG4SLib;
function g4s_cache_attend(ACache: PG4SCache; AState: PG4SPageState; ARows: Integer;
  ADevStarts: PInteger; ATokens: Integer; ADType: Integer; AQ: PG4SCacheView;
  ADevPool: Pointer; AKPlane: Integer; AVPlane: Integer; AScale: Single;
  AWindow: Integer; AOut: PG4SCacheView; ADevLse: PSingle): Integer; cdecl;
  external CG4SLib;

type
  { TGpuKvCache }
  TGpuKvCache = class(TBaseObject)
  private
    FHandle: PG4SCache;
    function Fail(const AStatus: Integer): Boolean;
  public
    destructor Destroy(); override;

    // g4s_cache_create: the whole workspace is allocated here
    function Open(const AGeometry: PG4SPageGeometry; const AConfig: PG4SCacheConfig;
      const AHipStream: Pointer = nil): Boolean;
    procedure Close();

    // one layer of a step: ADevStarts nil where every row has one token
    function Append(const AState: PG4SPageState; const ARows: Integer;
      const ADevStarts: PInteger; const ATokens: Integer; const ADType: Integer;
      const AQ: PG4SCacheView; const AK: PG4SCacheView; const AV: PG4SCacheView;
      const AQOut: PG4SCacheView; const ADevPositions: PInteger;
      const ADevFreqs: PSingle; const ADevPool: Pointer; const AKPlane: Integer;
      const AVPlane: Integer): Boolean;
    function Attend(const AState: PG4SPageState; const ARows: Integer;
      const ADevStarts: PInteger; const ATokens: Integer; const ADType: Integer;
      const AQ: PG4SCacheView; const ADevPool: Pointer; const AKPlane: Integer;
      const AVPlane: Integer; const AScale: Single; const AWindow: Integer;
      const AOut: PG4SCacheView; const ADevLse: PSingle = nil): Boolean;

    function LastError(): string;

    property Handle: PG4SCache read FHandle;
  end;

implementation

{ TGpuKvCache }

destructor TGpuKvCache.Destroy();
begin
  Close();
  inherited;
end;

function TGpuKvCache.LastError(): string;
begin
  Result := string(AnsiString(g4s_cache_last_error(FHandle)));
end;

function TGpuKvCache.Fail(const AStatus: Integer): Boolean;
begin
  GetErrors().Add(esError, CSM_ERR_CACHE, 'Cache status %d: %s', [AStatus, LastError()]);
  Result := False;
end;

function TGpuKvCache.Open(const AGeometry: PG4SPageGeometry; const AConfig: PG4SCacheConfig;
  const AHipStream: Pointer): Boolean;
var
  LStatus: Integer;
  LHandle: PG4SCache;
begin
  Close();
  LHandle := nil;
  LStatus := g4s_cache_create(@LHandle, AGeometry, AConfig, AHipStream);
  if LStatus <> G4S_OK then
    Exit(Fail(LStatus));
  FHandle := LHandle;
  Result := True;
end;

procedure TGpuKvCache.Close();
begin
  if FHandle <> nil then
  begin
    g4s_cache_destroy(FHandle);
    FHandle := nil;
  end;
end;

function TGpuKvCache.Append(const AState: PG4SPageState; const ARows: Integer;
  const ADevStarts: PInteger; const ATokens: Integer; const ADType: Integer;
  const AQ: PG4SCacheView; const AK: PG4SCacheView; const AV: PG4SCacheView;
  const AQOut: PG4SCacheView; const ADevPositions: PInteger; const ADevFreqs: PSingle;
  const ADevPool: Pointer; const AKPlane: Integer; const AVPlane: Integer): Boolean;
var
  LStatus: Integer;
begin
  LStatus := g4s_cache_append(FHandle, AState, ARows, ADevStarts, ATokens, ADType, AQ, AK, AV,
    AQOut, ADevPositions, ADevFreqs, ADevPool, AKPlane, AVPlane);
  if LStatus <> G4S_OK then
    Exit(Fail(LStatus));
  Result := True;
end;

function TGpuKvCache.Attend(const AState: PG4SPageState; const ARows: Integer;
  const ADevStarts: PInteger; const ATokens: Integer; const ADType: Integer;
  const AQ: PG4SCacheView; const ADevPool: Pointer; const AKPlane: Integer;
  const AVPlane: Integer; const AScale: Single; const AWindow: Integer;
  const AOut: PG4SCacheView; const ADevLse: PSingle): Boolean;
var
  LStatus: Integer;
begin
  LStatus := g4s_cache_attend(FHandle, AState, ARows, ADevStarts, ATokens, ADType, AQ, ADevPool,
    AKPlane, AVPlane, AScale, AWindow, AOut, ADevLse);
  if LStatus <> G4S_OK then
    Exit(Fail(LStatus));
  Result := True;
end;

end.
